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
// One entry's place; false when it is skipped.
__device__ __forceinline__ bool append_place(const dft_kv_append_args& a, int64_t i, int64_t& row, int64_t& page,
                                             int64_t& token) {
  const int64_t slot = ld_i(a.slots, i, a.slots_dtype);
  row = a.rows ? ld_i(a.rows, i, a.rows_dtype) : i;
  if (slot < 0 || row < 0) return false;
  page = slot / a.page_size;
  token = slot - page * a.page_size;
  if (page >= a.num_pages || row >= a.src_rows) {
    if (a.status) *a.status = 1;
    return false;
  }
  return true;
}

__global__ void __launch_bounds__(kThreads) kv_append_kernel(dft_kv_append_args a) {
  const int64_t width = (int64_t)a.heads * a.head_dim, total = a.n * width;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
    const int64_t i = e / width;
    const int c = (int)(e - i * width), h = c / a.head_dim, x = c - h * a.head_dim;
    int64_t row, page, token;
    if (!append_place(a, i, row, page, token)) continue;
    const float k = ld_f(a.k, row * a.k_row_stride + h * a.k_h_stride + x, a.src_dtype);
    const float v = ld_f(a.v, row * a.v_row_stride + h * a.v_h_stride + x, a.src_dtype);
    st_f(a.key_cache, page * a.kc_page_stride + token * a.kc_token_stride + h * a.kc_h_stride + x, a.cache_dtype, k);
    st_f(a.value_cache, page * a.vc_page_stride + token * a.vc_token_stride + h * a.vc_h_stride + x, a.cache_dtype, v);
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
  const int64_t total = a->n * a->heads * a->head_dim, blocks = (total + kThreads - 1) / kThreads;
  kv_append_kernel<<<(int)(blocks > 65536 ? 65536 : blocks), kThreads, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace dft
