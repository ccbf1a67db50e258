// dft_paged_attention: attention of new tokens over a paged cache.
//
// An item is 32 WM packed rows of one request and kv head over the keys they
// see, in tiles of 64.  The items' tiles form one line, cut into equal shares,
// one a workgroup: the requests' lengths, which only the device knows, neither
// leave workgroups idle nor set the grid.  A workgroup whose share holds an
// item whole writes its rows; one that holds a part writes the part's
// accumulators to the workspace, at most two parts a share, and a second
// launch joins them.  Where the block table is short the items are not cut.
//
// With few rows (decode: a token's group of heads) two waves take the halves
// of every tile, with more each wave takes rows of its own over whole tiles.
#include "attend.h"

namespace dft {
namespace {

using namespace attend;

constexpr int kCus = 256;
constexpr int kLeast = 4;      // tiles in a share
constexpr int kUncut = 8;      // an item of at most so many tiles is never cut
constexpr int kJoinWaves = 4;  // of the joining launch's workgroups

// What a share that begins inside an item leaves for the join.
struct Head {
  int64_t first, last, share;  // the item's tiles on the line, tiles per share
  int32_t b, g, tile, inside;
};

struct Plan {
  char* heads;
  float* parts;
  uint32_t magic;  // j / page_size = j * magic >> shift for j < 2^31
  int shift;
  int row_tiles;   // of the largest request there may be
  bool vec, uncut;
};

template <int D>
constexpr int part_floats() {  // of a wave's 32 rows: accumulators, reference, sum
  return 32 * D + 128;
}

struct Request {
  int64_t r0;
  int n, keys, before;  // rows, keys, keys in front of the rows' own (negative: some rows have none)
  int status;
};

__device__ __forceinline__ Request request(const dft_paged_attention_args& a, int b) {
  Request q;
  q.r0 = a.cu_seqlens ? a.cu_seqlens[b] : (int64_t)b * a.n_new;
  int64_t n = a.cu_seqlens ? (int64_t)a.cu_seqlens[b + 1] - q.r0 : a.n_new;
  q.status = n < 0 || n > a.n_new || q.r0 < 0 || q.r0 + n > a.rows ? DFT_STATUS_SPAN : 0;
  n = q.r0 < 0 ? 0 : min(min(n, (int64_t)a.n_new), a.rows - q.r0);
  q.n = (int)max(n, (int64_t)0);
  const int64_t top = 0x7fffffff - kTile, room = (int64_t)a.columns * a.page_size;
  const int64_t seq = max(ld_i(a.seq_len, b, a.seq_len_dtype), (int64_t)0);
  if (seq > room) q.status |= DFT_STATUS_TABLE;
  q.before = (int)(min(seq, top) - q.n);
  q.keys = a.num_pages ? (int)min(min(seq, room), top) : 0;
  return q;
}

// Tiles of the row tile's keys; one where it has none, so that its rows are written.
template <int BM>
__device__ __forceinline__ int tiles_of(const dft_paged_attention_args& a, const Request& q, int group, int tile) {
  int keys = q.keys;
  if (a.flags & DFT_ATTN_CAUSAL) {
    const int64_t end = min((int64_t)(tile + 1) * BM, (int64_t)q.n * group);
    keys = min(keys, q.before + (int)((end - 1) / group) + 1);
  }
  return max((keys + kTile - 1) / kTile, 1);
}

template <int BM>
__device__ __forceinline__ int row_tiles_of(const Request& q, int group) {
  return (int)(((int64_t)q.n * group + BM - 1) / BM);
}

// Sum of the threads' values in front of this thread's, and of all.
template <int NT>
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* red, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up(s, o);
    if (lane >= o) s += up;
  }
  if (lane == 63) red[wave] = s;
  __syncthreads();
  total = 0;
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) s += red[w];
    total += red[w];
  }
  return s - x;
}

// The rows of lane l's outputs
struct Place {
  int64_t row;
  int h;
  bool there;
};
__device__ __forceinline__ Place place_of(const Request& q, int group, int g, int64_t first) {
  const int64_t rows = (int64_t)q.n * group, p = min(first + (threadIdx.x & 31), rows - 1);
  const int64_t i = p / group;
  return {q.r0 + i, g * group + (int)(p - i * group), first + (threadIdx.x & 31) < rows};
}

template <int D, int WM, int WK, class T>
__global__ void __launch_bounds__(64 * WM * WK, D == 256 ? 1 : 2)
    paged_kernel(dft_paged_attention_args a, Scale sc, Plan pl) {
  constexpr int kRow = 2 * D, kBytes = kTile * kRow, NW = WM * WK, NT = 64 * NW, BM = 32 * WM, KW = kTile / WK;
  constexpr int kRows = 1024 / kRow, kCopies = kTile / (kRows * NW), kPieces = D / 8;
  typedef Rows<D, KW, T> Wave;
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  __shared__ __attribute__((aligned(1024))) char lds[2][2][kBytes];
  __shared__ char notes[NW][Wave::kNotes];
  __shared__ int ids[NW][2][kTile];                  // page ids of a tile's keys
  __shared__ u64x2 from[NW][kTile];                  // addresses of its keys and values
  __shared__ int64_t red[NW];
  __shared__ int spoiled;                            // the last tile found to hold a value that is not finite
  __shared__ int at_b, at_g, at_tile, at_off;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int wm = wave % WM, wk = wave / WM;
  const int group = a.hq / a.hkv;
  const bool causal = a.flags & DFT_ATTN_CAUSAL;

  // ---- this workgroup's share of the line
  int64_t pos, end, share = 0;
  int b, g, tile, off;
  if (pl.uncut) {
    const int64_t x = blockIdx.x;
    tile = (int)(x / ((int64_t)a.batch * a.hkv));
    const int pair = (int)(x - (int64_t)tile * a.batch * a.hkv);
    b = pair / a.hkv;
    g = pair - b * a.hkv;
    const Request q = request(a, b);
    if (a.status && tile == 0 && g == 0 && threadIdx.x == 0) a.status[b] = q.status;
    if (tile >= row_tiles_of<BM>(q, group)) return;
    pos = off = 0;
    end = tiles_of<BM>(a, q, group, tile);
  } else {
    const int per = (a.batch + NT - 1) / NT;
    const int b0 = min((int)threadIdx.x * per, a.batch), b1 = min(b0 + per, a.batch);
    auto weight = [&](int x) -> int64_t {  // of one kv head of request x
      const Request q = request(a, x);
      if (a.status && blockIdx.x == 0) a.status[x] = q.status;
      int64_t sum = 0;
      const int n = row_tiles_of<BM>(q, group);
      for (int t = 0; t < n; ++t) sum += tiles_of<BM>(a, q, group, t);
      return sum;
    };
    int64_t mine = 0, total;
    for (int x = b0; x < b1; ++x) mine += weight(x) * a.hkv;
    const int64_t ahead = scan<NT>(mine, red, total);
    share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)kLeast);
    pos = blockIdx.x * share;
    end = min(pos + share, total);
    if (pos >= ahead && pos < ahead + mine) {
      int64_t rest = pos - ahead, w = 0;
      int x = b0;
      for (; rest >= (w = weight(x)) * a.hkv; ++x) rest -= w * a.hkv;
      at_b = x;
      at_g = (int)(rest / w);
      rest -= at_g * w;
      const Request q = request(a, x);
      int t = 0;
      for (int n; rest >= (n = tiles_of<BM>(a, q, group, t)); ++t) rest -= n;
      at_tile = t;
      at_off = (int)rest;
    }
    __syncthreads();
    if (pos >= end) {
      if (threadIdx.x == 0) reinterpret_cast<Head*>(pl.heads)[blockIdx.x].inside = 0;
      return;
    }
    b = __builtin_amdgcn_readfirstlane(at_b);
    g = __builtin_amdgcn_readfirstlane(at_g);
    tile = __builtin_amdgcn_readfirstlane(at_tile);
    off = __builtin_amdgcn_readfirstlane(at_off);
    if (threadIdx.x == 0) {
      Head h;
      h.first = pos - off;
      h.last = h.first + tiles_of<BM>(a, request(a, b), group, tile);
      h.share = share;
      h.b = b, h.g = g, h.tile = tile, h.inside = off > 0;
      reinterpret_cast<Head*>(pl.heads)[blockIdx.x] = h;
    }
  }

  const uint32_t lds0 = lds_address(lds), ids0 = lds_address(ids[wave]);
  const int lrow = lane / kPieces, piece = lane % kPieces;
  Wave w;
  w.notes = lds_address(notes[wave]);

  while (true) {
    Request q = request(a, b);
    q.r0 = uniform64(q.r0);
    q.n = __builtin_amdgcn_readfirstlane(q.n);
    q.keys = __builtin_amdgcn_readfirstlane(q.keys);
    q.before = __builtin_amdgcn_readfirstlane(q.before);
    const int all = tiles_of<BM>(a, q, group, tile);
    const int begin = off, stop = (int)min((int64_t)all, off + (end - pos));
    const int64_t rows = (int64_t)q.n * group, pw = (int64_t)tile * BM + 32 * wm;
    const bool works = pw < rows;
    const Place to = place_of(q, group, g, min(pw, rows - 1));
    const int i = (int)(to.row - q.r0);
    const int fewest = a.anc_bits ? q.before  // keys that every row of the workgroup sees
                       : causal   ? min(q.before + (int)((int64_t)tile * BM / group) + 1, q.keys)
                                  : q.keys;
    uint64_t bits = 0;
    int limit = q.keys, least = q.keys, most = q.keys;  // keys the lane's row sees, all rows do, any does
    if (a.anc_bits) {
      bits = a.anc_bits[to.row];
      least = q.before;
    } else if (causal) {
      limit = min(q.before + i + 1, q.keys);
      least = __builtin_amdgcn_readlane(limit, 0), most = __builtin_amdgcn_readlane(limit, 31);
    }
    const int32_t* table = a.block_table + b * a.table_row_stride;
    const uint64_t kbase = (uint64_t)(uintptr_t)a.key_cache + 2 * (g * a.kc_h_stride);
    const uint64_t vbase = (uint64_t)(uintptr_t)a.value_cache + 2 * (g * a.vc_h_stride);

    // a key's page id, for every lane of this wave's own copy of the list
    auto fetch_ids = [&](int t) {
      const uint32_t j = (uint32_t)min(t * kTile + lane, q.keys - 1);
      const uint32_t col = (uint32_t)((uint64_t)j * pl.magic >> pl.shift);
      dma4_at((uint64_t)(uintptr_t)(table + col), ids0 + (t & 1) * 4 * kTile);
    };
    // the tile's keys and values; returns which of its keys there are
    auto copy = [&](int t, int stage) -> uint64_t {
      const int j = t * kTile + lane;
      const uint32_t jj = (uint32_t)min(j, q.keys - 1), col = (uint32_t)((uint64_t)jj * pl.magic >> pl.shift);
      const int id = ids[wave][t & 1][lane];
      const bool ok = j < q.keys && id >= 0 && id < a.num_pages;
      const int64_t page = ok ? id : 0, token = ok ? (int)(jj - col * a.page_size) : 0;
      u64x2 src = {kbase + 2 * (uint64_t)(page * a.kc_page_stride + token * a.kc_token_stride),
                   vbase + 2 * (uint64_t)(page * a.vc_page_stride + token * a.vc_token_stride)};
      from[wave][lane] = src;
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int x = 0; x < kCopies; ++x) {
        const int first = (x * NW + wave) * kRows, row = first + lrow;
        src = from[wave][row];
        const uint32_t at = lds0 + stage * 2 * kBytes + first * kRow;
        dma16_at(src[0] + ((piece ^ key_swizzle<D>(row)) << 4), at);
        dma16_at(src[1] + ((piece ^ value_swizzle<D>(row)) << 4), at + kBytes);
      }
      return __ballot(ok);
    };

    w.clear();
    if (q.keys > 0 && begin * kTile < q.keys) {
      if (threadIdx.x == 0) spoiled = -1;
      fetch_ids(begin);
      __builtin_amdgcn_s_waitcnt(kWaitDma);
      asm volatile("" ::: "memory");
      uint64_t there = copy(begin, begin & 1), next = 0;
      if (begin + 1 < stop) fetch_ids(begin + 1);
      w.load_q(static_cast<const uint16_t*>(a.q) + to.row * a.q_row_stride + to.h * a.q_h_stride, sc);
      for (int t = begin; t < stop; ++t, there = next) {
        __builtin_amdgcn_s_waitcnt(kWaitDma);
        __syncthreads();
        if (t + 1 < stop) {
          next = copy(t + 1, (t + 1) & 1);
          if (t + 2 < stop) fetch_ids(t + 2);
        }
        const int j0 = t * kTile + wk * KW;
        const uint32_t tile_at = lds0 + (t & 1) * 2 * kBytes, at = tile_at + wk * KW * kRow;
        const uint32_t slice = tile_at + kBytes + wave * (kBytes / NW);
        const uint64_t every = KW == 64 ? ~0ull : (1ull << KW) - 1, valid = there >> (wk * KW) & every;
        const bool acts = works && j0 < most, partial = valid != every || j0 + KW > least;
        uint64_t vis = every;
        if (partial) {
          if (a.anc_bits) {
            const int up = q.before - j0;
            vis = first_bits(up) | (up >= 64 || up <= -64 ? 0 : up >= 0 ? bits << up : bits >> -up);
          } else {
            vis = first_bits(limit - j0);
          }
          vis &= valid;
        }
        if (there != ~0ull || (t + 1) * kTile > fewest) {
          if (!finite<T, kBytes / NW>(slice)) spoiled = t;
          __syncthreads();
          if (spoiled == t) {
            if (acts) w.note(at + kBytes, vis);
            __syncthreads();
            clear_infinite<T, kBytes / NW>(slice);
            __syncthreads();
          }
        }
        if (acts) w.tile(at, at + kBytes, sc.c, partial, vis);
      }
      __syncthreads();
    }
    w.finish();

    if constexpr (WK == 2) {  // the halves of the tiles
      float* other = reinterpret_cast<float*>(&lds[0][0][0]);
      if (wk == 1) {
#pragma unroll
        for (int t = 0; t < Wave::DT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4*>(other + ((t * 4 + x) * 64 + lane) * 4) =
                f32x4{w.o[t][4 * x], w.o[t][4 * x + 1], w.o[t][4 * x + 2], w.o[t][4 * x + 3]};
        other[32 * D + lane] = w.top;
        other[32 * D + 64 + lane] = w.sum;
      }
      __syncthreads();
      if (wk == 0) {
        const float top = other[32 * D + lane], high = fmaxf(w.top, top);
        const float by = w.top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.top - high);
        const float his = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - high);
        w.top = high;
        w.sum = w.sum * by + other[32 * D + 64 + lane] * his;
#pragma unroll
        for (int t = 0; t < Wave::DT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const f32x4 y = *reinterpret_cast<f32x4*>(other + ((t * 4 + x) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) w.o[t][4 * x + e] = w.o[t][4 * x + e] * by + y[e] * his;
          }
      }
      __syncthreads();
    }

    if (works && wk == 0) {
      if (begin == 0 && stop == all) {
        const float sum = w.whole_sum(), by = weight_of(sum);
        if (to.there) {
          const int64_t out = to.row * a.o_row_stride + to.h * a.o_h_stride + 4 * half;
#pragma unroll
          for (int t = 0; t < Wave::DT; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              f32x4 y;
#pragma unroll
              for (int e = 0; e < 4; ++e) y[e] = w.o[t][4 * x + e] * by;
              store4(a.o, out + 32 * t + 8 * x, a.o_dtype, pl.vec, y);
            }
          if (a.lse && half == 0) a.lse[to.row * a.lse_row_stride + to.h] = lse_of(w.top, sum);
        }
      } else if (to.there) {
        float* part = pl.parts + (((int64_t)blockIdx.x * 2 + (begin == 0)) * WM + wm) * part_floats<D>();
#pragma unroll
        for (int t = 0; t < Wave::DT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4*>(part + ((t * 4 + x) * 64 + lane) * 4) =
                f32x4{w.o[t][4 * x], w.o[t][4 * x + 1], w.o[t][4 * x + 2], w.o[t][4 * x + 3]};
        part[32 * D + lane] = w.top;
        part[32 * D + 64 + lane] = w.sum;
      }
    }

    // the next item of the share
    pos += stop - begin;
    if (pos >= end) return;
    off = 0;
    if (++tile < row_tiles_of<BM>(q, group)) continue;
    tile = 0;
    if (++g < a.hkv) continue;
    g = 0;
    do {
      if (++b == a.batch) return;
    } while (__builtin_amdgcn_readfirstlane(request(a, b).n) == 0);
  }
}

// Joins the parts of the item that the share boundary in front of workgroup
// blockIdx.x cuts first: 32 columns of 32 rows, the parts dealt to the waves.
template <int D, int WM>
__global__ void __launch_bounds__(64 * kJoinWaves) join_kernel(dft_paged_attention_args a, Plan pl) {
  constexpr int BM = 32 * WM;
  const Head h = reinterpret_cast<const Head*>(pl.heads)[blockIdx.x];
  // cut elsewhere, or before: that boundary's workgroup joins it
  if (!h.inside || h.first < (int64_t)(blockIdx.x - 1) * h.share) return;
  __shared__ f32x4 sums[kJoinWaves][4][64];
  __shared__ float tops[kJoinWaves][64], totals[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int t = blockIdx.y % (D / 32), wm = blockIdx.y / (D / 32), group = a.hq / a.hkv;
  const Request q = request(a, h.b);
  const int64_t first = (int64_t)h.tile * BM + 32 * wm;
  if (first >= (int64_t)q.n * group) return;
  const Place to = place_of(q, group, h.g, first);
  const int64_t past = (h.last - 1) / h.share;  // the item's last share

  float top = -INFINITY, sum = 0;
  f32x4 o[4] = {};
  if (to.there)
    for (int64_t s = (int64_t)blockIdx.x - 1 + wave; s <= past; s += kJoinWaves) {
      const float* part = pl.parts + ((s * 2 + (s < blockIdx.x)) * WM + wm) * part_floats<D>();
      const float his = part[32 * D + lane], high = fmaxf(top, his);
      const float by = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - high);
      const float with = his == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(his - high);
      top = high;
      sum = sum * by + part[32 * D + 64 + lane] * with;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        o[x] = o[x] * by + *reinterpret_cast<const f32x4*>(part + ((t * 4 + x) * 64 + lane) * 4) * with;
    }
  tops[wave][lane] = top;
  totals[wave][lane] = sum;
#pragma unroll
  for (int x = 0; x < 4; ++x) sums[wave][x][lane] = o[x];
  __syncthreads();
  if (wave) return;
  float high = top;
  for (int s = 1; s < kJoinWaves; ++s) high = fmaxf(high, tops[s][lane]);
  sum = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) o[x] = f32x4{};
  for (int s = 0; s < kJoinWaves; ++s) {
    const float by = tops[s][lane] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(tops[s][lane] - high);
    sum += totals[s][lane] * by;
#pragma unroll
    for (int x = 0; x < 4; ++x) o[x] += sums[s][x][lane] * by;
  }
  sum += __shfl_xor(sum, 32);
  if (!to.there) return;
  const float by = weight_of(sum);
  const int64_t out = to.row * a.o_row_stride + to.h * a.o_h_stride + 32 * t + 4 * half;
#pragma unroll
  for (int x = 0; x < 4; ++x) store4(a.o, out + 8 * x, a.o_dtype, pl.vec, o[x] * by);
  if (a.lse && t == 0 && half == 0) a.lse[to.row * a.lse_row_stride + to.h] = lse_of(high, sum);
}

// The launch's sizes.
struct Shape {
  int wm;
  bool uncut;
  int64_t grid, heads_bytes, parts_bytes;
};
Shape shape_of(const dft_paged_attention_args& a) {
  Shape s;
  const int64_t rows = (int64_t)a.n_new * (a.hq / a.hkv);
  s.wm = rows <= 32 ? 1 : 4;
  s.uncut = (int64_t)a.columns * a.page_size <= kUncut * kTile;
  if (s.uncut) {
    s.grid = (int64_t)a.batch * a.hkv * ((rows + 32 * s.wm - 1) / (32 * s.wm));
    s.heads_bytes = s.parts_bytes = 0;
    return s;
  }
  // as many workgroups as the LDS holds: 512 D bytes of tiles each, and a little
  s.grid = kCus * (a.head_dim == 256 ? 1 : a.head_dim == 128 ? 2 : 4);
  s.heads_bytes = s.grid * sizeof(Head);
  s.parts_bytes = s.grid * 2 * s.wm * (32 * a.head_dim + 128) * sizeof(float);
  return s;
}

template <int D, int WM, int WK, class T>
int launch(const dft_paged_attention_args& a, const Shape& s, const Plan& pl, hipStream_t stream) {
  paged_kernel<D, WM, WK, T><<<(unsigned)s.grid, 64 * WM * WK, 0, stream>>>(a, split_scale(a.scale), pl);
  if (hipGetLastError() != hipSuccess) return DFT_ERR_LAUNCH;
  if (s.uncut) return DFT_OK;
  join_kernel<D, WM><<<dim3((unsigned)s.grid, WM * D / 32), 64 * kJoinWaves, 0, stream>>>(a, pl);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

template <int D, class T>
int launch_rows(const dft_paged_attention_args& a, const Shape& s, const Plan& pl, hipStream_t stream) {
  return s.wm == 1 ? launch<D, 1, 2, T>(a, s, pl, stream) : launch<D, 4, 1, T>(a, s, pl, stream);
}

template <class T>
int launch_type(const dft_paged_attention_args& a, const Shape& s, const Plan& pl, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch_rows<64, T>(a, s, pl, stream);
    case 128: return launch_rows<128, T>(a, s, pl, stream);
    default: return launch_rows<256, T>(a, s, pl, stream);
  }
}

}  // namespace

int64_t paged_attention_workspace(const dft_paged_attention_args* a) {
  const Shape s = shape_of(*a);
  return s.heads_bytes + s.parts_bytes;
}

int launch_paged_attention(const dft_paged_attention_args* a, hipStream_t stream) {
  const Shape s = shape_of(*a);
  if (s.grid > 0xffffffffll / 256) return DFT_ERR_UNSUPPORTED;  // a grid counts work-items in 32 bits
  Plan pl = {};
  pl.heads = static_cast<char*>(a->workspace);
  pl.parts = reinterpret_cast<float*>(pl.heads + s.heads_bytes);
  int log = 0;
  while ((1ll << log) < a->page_size) ++log;
  pl.shift = 31 + log;
  pl.magic = (uint32_t)(((1ull << pl.shift) + a->page_size - 1) / a->page_size);
  pl.row_tiles = 0;
  pl.vec = vector_out(*a);
  pl.uncut = s.uncut;
  return a->dtype == DFT_BF16 ? launch_type<Bf16>(*a, s, pl, stream) : launch_type<F16>(*a, s, pl, stream);
}

}  // namespace dft
