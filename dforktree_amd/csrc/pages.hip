// The paged KV cache of the full-attention layers:
//   dft_page_plan   block tables, slot maps and positions from the requests'
//                   lengths, pages taken from and returned to a ring
//   dft_kv_append   new K/V rows (or an accepted path's) into their slots
//
// Neither computes: the plan is bound by launch latency up to some ten
// thousand rows, then by the 16 bytes it writes per row; the append by HBM.
#include <stdint.h>

#include "dft_device.h"

namespace dft {
namespace {

constexpr int kThreads = 256;

// ---- page plan -------------------------------------------------------------
// Every workgroup scans the batch's lengths itself (three running sums over
// at most 8192 requests: rows, pages taken, pages returned), so one launch
// suffices; what is per row and per page is then dealt out over the grid.
struct Sums {
  int64_t v[2];
};

// Exclusive scan over the block of two sums per thread.
__device__ __forceinline__ Sums block_scan(Sums x, int64_t (*red)[kThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Sums s = x;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t up = __shfl_up(s.v[k], o);
      if (lane >= o) s.v[k] += up;
    }
    if (lane == 63) red[k][wave] = s.v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int64_t before = 0;
    for (int w = 0; w < wave; ++w) before += red[k][w];
    s.v[k] += before - x.v[k];
  }
  __syncthreads();
  return s;
}

__device__ __forceinline__ int32_t clip32(int64_t v) { return (int32_t)(v < 0x7fffffffll ? v : 0x7fffffffll); }

// The first request whose running sum `end` exceeds i.
__device__ __forceinline__ int find(const int32_t* end, int batch, int64_t i) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)end[mid] > i)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) page_plan_kernel(dft_page_plan_args a) {
  extern __shared__ int32_t shared[];
  __shared__ int64_t red[2][kThreads / 64];
  const int B = a.batch, ps = a.page_size;
  int32_t* end = shared;            // rows up to and with each request
  int32_t* take = shared + B;       // pages taken up to and with it
  int32_t* give = shared + 2 * B;   // pages returned
  int32_t* state = shared + 3 * B;  // its status word
  const int64_t head = a.free_pos[0], tail = a.free_pos[1];
  const int64_t free_now = min(max(tail - head, (int64_t)0), a.capacity);
  const int per = (B + kThreads - 1) / kThreads;
  const int b0 = min((int)threadIdx.x * per, B), b1 = min(b0 + per, B);

  // rows
  Sums s = {{0, 0}};
  for (int b = b0; b < b1; ++b) s.v[0] += max(ld_i(a.new_len, b, a.new_len_dtype), (int64_t)0);
  s = block_scan(s, red);
  for (int b = b0; b < b1; ++b) {
    s.v[0] += max(ld_i(a.new_len, b, a.new_len_dtype), (int64_t)0);
    end[b] = (int32_t)min(s.v[0], a.rows);
  }
  __syncthreads();
  // pages
  auto pages = [&](int b, int& status, int64_t& prefix, int& n) -> int64_t {  // wanted - held
    const int64_t len = ld_i(a.new_len, b, a.new_len_dtype), pre = ld_i(a.prefix_len, b, a.prefix_len_dtype);
    n = end[b] - (b ? end[b - 1] : 0);
    prefix = max(pre, (int64_t)0);
    status = n != len || pre < 0 ? DFT_STATUS_SPAN : 0;
    const int64_t want = (prefix + n + ps - 1) / ps;
    if (want > a.columns) status |= DFT_STATUS_TABLE;
    return want - min(max(a.held[b], 0), a.columns);
  };
  int status, n;
  int64_t prefix;
  s = {{0, 0}};
  for (int b = b0; b < b1; ++b) {
    const int64_t d = pages(b, status, prefix, n);
    if (!(status & DFT_STATUS_TABLE)) {
      s.v[0] += max(d, (int64_t)0);
      if (a.trim) s.v[1] += max(-d, (int64_t)0);
    }
  }
  s = block_scan(s, red);
  for (int b = b0; b < b1; ++b) {
    const int64_t d = pages(b, status, prefix, n);
    if (!(status & DFT_STATUS_TABLE)) {
      s.v[0] += max(d, (int64_t)0);
      if (a.trim) s.v[1] += max(-d, (int64_t)0);
      if ((d > 0 && s.v[0] > free_now) || (a.trim && d < 0 && s.v[1] > a.capacity - free_now))
        status |= DFT_STATUS_PAGES;
    }
    take[b] = clip32(s.v[0]);
    give[b] = clip32(s.v[1]);
    state[b] = status;
    if (blockIdx.x == 0) {
      const bool served = !(status & (DFT_STATUS_TABLE | DFT_STATUS_PAGES));
      const int held = min(max(a.held[b], 0), a.columns);
      a.status[b] = status;
      a.cu_seqlens[b + 1] = end[b];
      a.seq_len[b] = served ? (int32_t)(prefix + n) : 0;
      a.held_out[b] = served && (d > 0 || a.trim) ? (int32_t)(held + d) : held;
    }
  }
  __syncthreads();
  // What is served of a running sum with an upper bound are its first
  // entries, those without a refused one in front: `served` of it.
  auto served_of = [&](const int32_t* sum, int64_t limit) -> int64_t {
    int lo = 0, hi = B;  // requests whose sum is within the limit
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)sum[mid] > limit)
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo ? sum[lo - 1] : 0;
  };
  const int64_t taken = B ? served_of(take, free_now) : 0, given = B ? served_of(give, a.capacity - free_now) : 0;
  const int64_t rows = B ? end[B - 1] : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.cu_seqlens[0] = 0;
    a.free_pos_out[0] = head + taken;
    a.free_pos_out[1] = tail + given;
  }

  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  auto ring = [&](int64_t i) -> int64_t {  // i >= 0 in a valid ring; any i stays inside
    const int64_t r = i % a.capacity;
    return r < 0 ? r + a.capacity : r;
  };
  for (int64_t p = first; p < taken; p += step) {
    const int b = find(take, B, p);
    const int held = min(max(a.held[b], 0), a.columns);
    const int64_t col = held + p - (b ? take[b - 1] : 0);
    a.block_table[b * a.table_row_stride + col] = a.free_pages[ring(head + p)];
  }
  for (int64_t p = first; p < given; p += step) {
    const int b = find(give, B, p);
    const int64_t want = (max(ld_i(a.prefix_len, b, a.prefix_len_dtype), (int64_t)0) + end[b] -
                          (b ? end[b - 1] : 0) + ps - 1) / ps;
    const int64_t col = want + p - (b ? give[b - 1] : 0);
    a.free_pages[ring(tail + p)] = a.block_table[b * a.table_row_stride + col];
  }
  for (int64_t r = first; r < a.rows; r += step) {
    int64_t slot = -1, at = 0;
    if (r < rows) {
      const int b = find(end, B, r);
      const int64_t pre = max(ld_i(a.prefix_len, b, a.prefix_len_dtype), (int64_t)0);
      const int64_t place = pre + r - (b ? end[b - 1] : 0);
      at = a.depth ? pre + ld_i(a.depth, r, a.depth_dtype) : place;
      if (!(state[b] & (DFT_STATUS_TABLE | DFT_STATUS_PAGES))) {
        const int held = min(max(a.held[b], 0), a.columns);
        const int64_t col = place / ps;
        // a new page's id comes from the ring: another workgroup writes its cell
        const int32_t page = col < held ? a.block_table[b * a.table_row_stride + col]
                                        : a.free_pages[ring(head + (b ? take[b - 1] : 0) + col - held)];
        if (page >= 0) slot = (int64_t)page * ps + place % ps;
      }
    }
    st_i(a.slots, r, a.index_dtype, slot);
    st_i(a.positions, r, a.index_dtype, at);
  }
}

// ---- KV append -------------------------------------------------------------
struct Append {
  uint32_t magic;     // slot / page_size = slot * magic >> shift for slot < 2^31
  int shift;
  int pieces, log;    // of an entry; log2 of the threads on an entry
  int per_head;       // pieces of a head
};

// An entry's place; false when it is skipped.
__device__ __forceinline__ bool append_place(const dft_kv_append_args& a, const Append& p, int64_t i, int64_t& row,
                                             int64_t& page, int64_t& token) {
  const int64_t slot = ld_i(a.slots, i, a.slots_dtype);
  row = a.rows ? ld_i(a.rows, i, a.rows_dtype) : i;
  if (slot < 0 || row < 0) return false;
  page = slot <= 0x7fffffffll ? (int64_t)((uint64_t)(uint32_t)slot * p.magic >> p.shift) : slot / a.page_size;
  token = slot - page * a.page_size;
  if (page >= a.num_pages || row >= a.src_rows) {
    if (a.status) *a.status = 1;
    return false;
  }
  return true;
}

// Eight elements, cast; of one type they keep their bits.
template <int SRC, int DST>
__device__ __forceinline__ void append_piece(const void* src, int64_t from, void* dst, int64_t to) {
  if constexpr (SRC == DST && SRC != DFT_F32) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(dst) + to) =
        *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(src) + from);
  } else if constexpr (SRC == DST) {
    const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const float*>(src) + from);
    u32x4* d = reinterpret_cast<u32x4*>(static_cast<float*>(dst) + to);
    const u32x4 lo = s[0], hi = s[1];
    d[0] = lo;
    d[1] = hi;
  } else {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    f32x8 x;
    if constexpr (SRC == DFT_BF16)
      x = __builtin_convertvector(*reinterpret_cast<const bf16x8*>(static_cast<const uint16_t*>(src) + from), f32x8);
    else if constexpr (SRC == DFT_F16)
      x = __builtin_convertvector(*reinterpret_cast<const f16x8*>(static_cast<const uint16_t*>(src) + from), f32x8);
    else
      x = *reinterpret_cast<const f32x8*>(static_cast<const float*>(src) + from);
    if constexpr (DST == DFT_BF16)
      *reinterpret_cast<bf16x8*>(static_cast<uint16_t*>(dst) + to) = __builtin_convertvector(x, bf16x8);
    else if constexpr (DST == DFT_F16)
      *reinterpret_cast<f16x8*>(static_cast<uint16_t*>(dst) + to) = __builtin_convertvector(x, f16x8);
    else
      *reinterpret_cast<f32x8*>(static_cast<float*>(dst) + to) = x;
  }
}

// 2^log threads take an entry, each a piece of eight elements (or several) of
// its key and its value; a thread's head and column are the same for every
// entry.
template <int SRC, int DST>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(dft_kv_append_args a, Append p) {
  const int lane = threadIdx.x & ((1 << p.log) - 1), per = kThreads >> p.log;
  for (int piece = lane; piece < p.pieces; piece += 1 << p.log) {
    const int h = piece / p.per_head, x = 8 * (piece - h * p.per_head);
    const int64_t ks = h * a.k_h_stride + x, vs = h * a.v_h_stride + x, kd = h * a.kc_h_stride + x, vd = h * a.vc_h_stride + x;
#pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * per + (threadIdx.x >> p.log); i < a.n; i += (int64_t)gridDim.x * per) {
      int64_t row, page, token;
      if (!append_place(a, p, i, row, page, token)) continue;
      append_piece<SRC, DST>(a.k, row * a.k_row_stride + ks, a.key_cache,
                             page * a.kc_page_stride + token * a.kc_token_stride + kd);
      append_piece<SRC, DST>(a.v, row * a.v_row_stride + vs, a.value_cache,
                             page * a.vc_page_stride + token * a.vc_token_stride + vd);
    }
  }
}

// Rows without 16-byte pieces: element by element.
__global__ void __launch_bounds__(kThreads) kv_append_elements_kernel(dft_kv_append_args a, Append p) {
  const int64_t width = (int64_t)a.heads * a.head_dim, total = a.n * width;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
    const int64_t i = e / width;
    const int c = (int)(e - i * width), h = c / a.head_dim, x = c - h * a.head_dim;
    int64_t row, page, token;
    if (!append_place(a, p, i, row, page, token)) continue;
    const int64_t ks = row * a.k_row_stride + h * a.k_h_stride + x, vs = row * a.v_row_stride + h * a.v_h_stride + x;
    const int64_t kd = page * a.kc_page_stride + token * a.kc_token_stride + h * a.kc_h_stride + x;
    const int64_t vd = page * a.vc_page_stride + token * a.vc_token_stride + h * a.vc_h_stride + x;
    if (a.src_dtype == a.cache_dtype && a.src_dtype != DFT_F32) {  // of one type: the bits
      static_cast<uint16_t*>(a.key_cache)[kd] = static_cast<const uint16_t*>(a.k)[ks];
      static_cast<uint16_t*>(a.value_cache)[vd] = static_cast<const uint16_t*>(a.v)[vs];
    } else {
      st_f(a.key_cache, kd, a.cache_dtype, ld_f(a.k, ks, a.src_dtype));
      st_f(a.value_cache, vd, a.cache_dtype, ld_f(a.v, vs, a.src_dtype));
    }
  }
}

template <int SRC>
void launch_append(const dft_kv_append_args& a, const Append& p, int grid, hipStream_t stream) {
  switch (a.cache_dtype) {
    case DFT_BF16: kv_append_kernel<SRC, DFT_BF16><<<grid, kThreads, 0, stream>>>(a, p); break;
    case DFT_F16: kv_append_kernel<SRC, DFT_F16><<<grid, kThreads, 0, stream>>>(a, p); break;
    default: kv_append_kernel<SRC, DFT_F32><<<grid, kThreads, 0, stream>>>(a, p); break;
  }
}

}  // namespace

int launch_page_plan(const dft_page_plan_args* a, hipStream_t stream) {
  const int64_t blocks = (a->rows + 1023) / 1024;
  const int grid = (int)(blocks < 1 ? 1 : blocks > 512 ? 512 : blocks);
  const size_t lds = 4 * sizeof(int32_t) * (size_t)a->batch;
  if (lds > 48 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(page_plan_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          (int)lds) != hipSuccess)
    return DFT_ERR_LAUNCH;
  page_plan_kernel<<<grid, kThreads, lds, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

int launch_kv_append(const dft_kv_append_args* a, hipStream_t stream) {
  Append p = {};
  int log = 0;
  while ((1ll << log) < a->page_size) ++log;
  p.shift = 31 + log;
  p.magic = (uint32_t)(((1ull << p.shift) + a->page_size - 1) / a->page_size);
  // pieces of eight elements: 16-byte aligned addresses and strides (32 for fp32, which only a vector of its own needs)
  auto aligned = [](const void* q, int dt, int64_t s0, int64_t s1, int64_t s2) {
    return reinterpret_cast<uintptr_t>(q) % (dt == DFT_F32 ? 32 : 16) == 0 && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0;
  };
  const bool pieces = a->head_dim % 8 == 0 && aligned(a->k, a->src_dtype, a->k_row_stride, a->k_h_stride, 0) &&
                      aligned(a->v, a->src_dtype, a->v_row_stride, a->v_h_stride, 0) &&
                      aligned(a->key_cache, a->cache_dtype, a->kc_page_stride, a->kc_token_stride, a->kc_h_stride) &&
                      aligned(a->value_cache, a->cache_dtype, a->vc_page_stride, a->vc_token_stride, a->vc_h_stride) &&
                      (int64_t)a->heads * a->head_dim < 0x7fffffff;
  if (!pieces) {
    const int64_t total = a->n * a->heads * a->head_dim, blocks = (total + kThreads - 1) / kThreads;
    kv_append_elements_kernel<<<(int)(blocks > 65536 ? 65536 : blocks), kThreads, 0, stream>>>(*a, p);
    return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
  }
  p.per_head = a->head_dim / 8;
  p.pieces = a->heads * p.per_head;
  while ((1 << p.log) < p.pieces && (1 << p.log) < kThreads) ++p.log;
  // up to four entries a thread where that still leaves sixteen workgroups a CU
  const int64_t entries = kThreads >> p.log, all = (a->n + entries - 1) / entries;
  const int64_t blocks = all <= 4096 ? all : all / 4 > 4096 ? all / 4 : 4096;
  const int grid = (int)(blocks > (1 << 20) ? (1 << 20) : blocks);
  switch (a->src_dtype) {
    case DFT_BF16: launch_append<DFT_BF16>(*a, p, grid, stream); break;
    case DFT_F16: launch_append<DFT_F16>(*a, p, grid, stream); break;
    default: launch_append<DFT_F32>(*a, p, grid, stream); break;
  }
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace dft
