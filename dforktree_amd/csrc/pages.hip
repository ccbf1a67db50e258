// The paged KV cache of the full-attention layers:
//   dft_page_plan   block tables, slot maps and positions from the requests'
//                   lengths, pages taken from and returned to a ring
//   dft_kv_append   new K/V rows (or an accepted path's) into their slots
//
// Neither computes: the plan is bound by the latency of its look-ups (5.6 us
// for 64 requests, 7.1 for 4608 rows of 128, 11.9 for 256000 of 1000), the append
// by HBM (16387 rows of 8 heads x 128: 21.6 us, 6.2 TB/s).
#include <stdint.h>

#include "dft_device.h"

namespace dft {
namespace {

constexpr int kThreads = 256;

// ---- page plan -------------------------------------------------------------
// Every workgroup scans the batch's lengths itself (running sums over at most
// 8192 requests: rows, then pages taken and returned), so one launch suffices;
// what is per row and per page is then dealt out over the grid, a row a
// thread: a row's look-ups (its request, its page) follow each other, so the
// time is their latency and the rows that a thread takes.  Divisions are by
// multiplication while they fit 31 bits.
struct PagePlan {
  uint32_t magic, ring_magic;  // x / page_size = x * magic >> shift for x < 2^31; the same by capacity
  int shift, ring_shift;
};

struct Sums {
  int64_t v[2];
};

// Exclusive scan over the block of two sums per thread.
template <int THREADS>
__device__ __forceinline__ Sums block_scan(Sums x, int64_t (*red)[THREADS / 64]) {
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

template <int THREADS>
__global__ void __launch_bounds__(THREADS) page_plan_kernel(dft_page_plan_args a, PagePlan p) {
  extern __shared__ int32_t shared[];
  __shared__ int64_t red[2][THREADS / 64];
  __shared__ int32_t within[2];  // the sums served: of pages taken, of pages returned
  const int B = a.batch, ps = a.page_size;
  int32_t* end = shared;            // rows up to and with each request
  int32_t* take = shared + B;       // pages taken up to and with it
  int32_t* give = shared + 2 * B;   // pages returned
  int32_t* state = shared + 3 * B;  // its status word
  const int64_t head = a.free_pos[0], tail = a.free_pos[1];
  const int64_t free_now = min(max(tail - head, (int64_t)0), a.capacity);
  const int per = (B + THREADS - 1) / THREADS;
  const int b0 = min((int)threadIdx.x * per, B), b1 = min(b0 + per, B);
  auto over = [&](int64_t x) -> int64_t {  // x / page_size
    return x <= 0x7fffffffll ? (int64_t)((uint64_t)(uint32_t)x * p.magic >> p.shift) : x / ps;
  };

  // Lengths as far as they matter, so that no sum of them leaves 64 bits: a
  // prefix past kFar needs more pages than a table has columns (2^31) even of
  // the largest pages (2^31), more new tokens than `rows` are cut to it.
  constexpr int64_t kFar = INT64_MAX - (1ll << 33);
  auto prefix_of = [&](int b) { return min(max(ld_i(a.prefix_len, b, a.prefix_len_dtype), (int64_t)0), kFar); };
  auto new_of = [&](int b) { return min(max(ld_i(a.new_len, b, a.new_len_dtype), (int64_t)0), a.rows + 1); };

  // rows
  if (threadIdx.x < 2) within[threadIdx.x] = 0;
  Sums s = {{0, 0}};
  for (int b = b0; b < b1; ++b) s.v[0] += new_of(b);
  s = block_scan<THREADS>(s, red);
  for (int b = b0; b < b1; ++b) {
    s.v[0] += new_of(b);
    end[b] = (int32_t)min(s.v[0], a.rows);
  }
  __syncthreads();
  // pages
  auto pages = [&](int b, int& status, int64_t& prefix, int& n) -> int64_t {  // wanted - held
    const int64_t len = ld_i(a.new_len, b, a.new_len_dtype), pre = ld_i(a.prefix_len, b, a.prefix_len_dtype);
    n = end[b] - (b ? end[b - 1] : 0);
    prefix = min(max(pre, (int64_t)0), kFar);
    status = n != len || pre < 0 ? DFT_STATUS_SPAN : 0;
    const int64_t want = over(prefix + n + ps - 1);
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
  s = block_scan<THREADS>(s, red);
  const int64_t room = a.capacity - free_now;
  for (int b = b0; b < b1; ++b) {
    const int64_t d = pages(b, status, prefix, n);
    if (!(status & DFT_STATUS_TABLE)) {
      s.v[0] += max(d, (int64_t)0);
      if (a.trim) s.v[1] += max(-d, (int64_t)0);
      if ((d > 0 && s.v[0] > free_now) || (a.trim && d < 0 && s.v[1] > room)) status |= DFT_STATUS_PAGES;
    }
    take[b] = clip32(s.v[0]);
    give[b] = clip32(s.v[1]);
    state[b] = status;
    if (blockIdx.x == 0) {
      const bool served = !(status & (DFT_STATUS_TABLE | DFT_STATUS_PAGES));
      const int held = min(max(a.held[b], 0), a.columns);
      a.status[b] = status;
      a.cu_seqlens[b + 1] = end[b];
      a.seq_len[b] = served ? clip32(prefix + n) : 0;
      a.held_out[b] = served && (d > 0 || a.trim) ? (int32_t)(held + d) : held;
    }
  }
  __syncthreads();
  // What is served of a running sum with an upper bound are its first
  // entries, those without a refused one in front: the last within it.
  for (int b = b0; b < b1; ++b) {
    if (take[b] <= free_now && (b + 1 == B || take[b + 1] > free_now)) within[0] = take[b];
    if (give[b] <= room && (b + 1 == B || give[b + 1] > room)) within[1] = give[b];
  }
  __syncthreads();
  const int64_t taken = within[0], given = within[1];
  const int64_t rows = B ? end[B - 1] : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.cu_seqlens[0] = 0;
    a.free_pos_out[0] = head + taken;
    a.free_pos_out[1] = tail + given;
  }

  // cells of the ring, `ahead` (at most its capacity) behind its first or its last
  auto wrap = [&](int64_t i) { return i >= a.capacity ? i - a.capacity : i; };
  auto cell = [&](int64_t i) -> int64_t {
    if (i >= 0 && i <= 0x7fffffffll) return i - (int64_t)((uint64_t)i * p.ring_magic >> p.ring_shift) * a.capacity;
    const int64_t r = i % a.capacity;
    return r < 0 ? r + a.capacity : r;
  };
  const int64_t front = cell(head), back = cell(tail);
  const int64_t step = (int64_t)gridDim.x * THREADS, first = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  // pages from the grid's other end: the last threads have the fewest rows
  const int64_t turned = step - 1 - first;
  for (int64_t x = turned; x < taken; x += step) {
    const int b = find(take, B, x);
    const int held = min(max(a.held[b], 0), a.columns);
    const int64_t col = held + x - (b ? take[b - 1] : 0);
    a.block_table[b * a.table_row_stride + col] = a.free_pages[wrap(front + x)];
  }
  for (int64_t x = turned; x < given; x += step) {
    const int b = find(give, B, x);
    const int64_t want = over(prefix_of(b) + end[b] - (b ? end[b - 1] : 0) + ps - 1);
    const int64_t col = want + x - (b ? give[b - 1] : 0);
    a.free_pages[wrap(back + x)] = a.block_table[b * a.table_row_stride + col];
  }
  for (int64_t r = first; r < a.rows; r += step) {
    int64_t slot = -1, at = 0;
    if (r < rows) {
      const int b = find(end, B, r);
      const int64_t pre = prefix_of(b);
      const int64_t place = pre + r - (b ? end[b - 1] : 0);
      at = a.depth ? pre + ld_i(a.depth, r, a.depth_dtype) : place;
      if (!(state[b] & (DFT_STATUS_TABLE | DFT_STATUS_PAGES))) {
        const int held = min(max(a.held[b], 0), a.columns);
        const int64_t col = over(place);
        // a new page's id comes from the ring: another workgroup writes its cell
        const int32_t page = col < held ? a.block_table[b * a.table_row_stride + col]
                                        : a.free_pages[wrap(front + (b ? take[b - 1] : 0) + col - held)];
        if (page >= 0) slot = (int64_t)page * ps + (place - col * ps);
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
  PagePlan p;
  page_magic(a->page_size, p.magic, p.shift);
  page_magic((int)a->capacity, p.ring_magic, p.ring_shift);
  // a request a thread as far as a workgroup goes
  const bool wide = a->batch > 256;
  const int threads = wide ? 1024 : 256;
  const int64_t blocks = (a->rows + a->rows / a->page_size + a->batch + threads - 1) / threads;
  const int most = wide ? 256 : 1024;  // all at work at once
  const int grid = (int)(blocks < 1 ? 1 : blocks > most ? most : blocks);
  const size_t lds = 4 * sizeof(int32_t) * (size_t)a->batch;
  if (lds > 48 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(page_plan_kernel<1024>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return DFT_ERR_LAUNCH;
  if (wide)
    page_plan_kernel<1024><<<grid, 1024, lds, stream>>>(*a, p);
  else
    page_plan_kernel<256><<<grid, 256, lds, stream>>>(*a, p);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

int launch_kv_append(const dft_kv_append_args* a, hipStream_t stream) {
  Append p = {};
  page_magic(a->page_size, p.magic, p.shift);
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
