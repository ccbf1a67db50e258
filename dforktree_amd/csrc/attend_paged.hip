// dft_paged_attention: attention of new tokens over a paged cache.
//
// An item is a tile of packed rows of one request (row p: token p / group,
// head p % group of a kv head) over the keys they see, in tiles.  A kv head's
// items stand in one line of key tiles, cut into equal shares, one a
// workgroup: the requests' lengths, which only the device knows, neither leave
// workgroups idle nor set the grid.  The kv heads' lines are cut alike, and
// their workgroups run side by side: one token's heads, which lie together,
// are read at about the same time.  A workgroup whose share holds an item
// whole writes its rows; one that holds a part writes the part's accumulators
// to the workspace, at most two parts a share, and a second launch joins them.
// Where the block table is short the items are not cut.
//
// few_kernel: up to 32 rows in all (decode: a token's group of heads), bound
// by the cache's bytes.  many_kernel: more rows, 32 a wave.
#include "attend.h"

namespace dft {
namespace {

using namespace attend;

constexpr int kCus = 256, kXcds = 8;
// Keys in a share at least.  With few rows a part costs little, and a short
// cache is read sooner by more workgroups (one request of 1000 keys, 8 kv
// heads, d 128: 16.7 us a step of 64, 21.9 of 256); with many its accumulators
// cost more than that (a tree of 32 nodes over 8000 keys: 38.2 and 33.8 us).
constexpr int kLeastFew = 64, kLeastMany = 256;
// Where the whole table holds at most so many keys no item is cut: no scan, no
// parts, no second launch.  470 keys each in a table of 496, uncut, and in one
// of 640, cut (8 kv heads, d 128), us a call: one token for 1, 4, 16 and 64
// requests 18.1, 18.3, 18.6, 27.3 and 16.0, 18.8, 22.7, 30.5; trees of 32 nodes
// 19.9, 19.9, 21.9, 41.7 and 27.3, 28.3, 32.4, 44.1.  (A single request's token
// alone is read sooner by more workgroups.)
constexpr int kUncutKeys = 512;

// What a share that begins inside an item leaves for the join.
struct Head {
  int64_t first, last, share;  // the item's tiles on the line, tiles per share
  int32_t b, tile, inside, pad;
};

struct Plan {
  char* heads;
  float* parts;
  uint32_t magic;  // j / page_size = j * magic >> shift for j < 2^31
  int shift;
  int shares;      // of a kv head's line
  bool vec, uncut;
};

// A part in the workspace: units of 64 lanes x 4 accumulators, then every
// row's reference and sum.
template <int D, int BM>
constexpr int part_floats() {
  return BM * (D + 2);
}

struct Request {
  int64_t r0;
  int n, keys;  // rows (times the group within 31 bits), keys
  int before;   // keys in front of the first row's own (negative: some rows have none)
  int status;
};

// How a request's lengths are read: by each lane for itself, or once for the
// wave, from arrays that this launch does not write.
struct ByLane {
  static __device__ __forceinline__ int i32(const int32_t* p) { return *p; }
  static __device__ __forceinline__ int64_t index(const void* p, int64_t i, int dt) { return ld_i(p, i, dt); }
};
struct ByWave {
  typedef const __attribute__((address_space(4))) int32_t* Words;
  static __device__ __forceinline__ int i32(const int32_t* p) { return *(Words)(uintptr_t)p; }
  static __device__ __forceinline__ int64_t index(const void* p, int64_t i, int dt) {
    const Words w = (Words)(uintptr_t)p;
    const bool wide = dt == DFT_I64;
    const int lo = w[wide ? 2 * i : i], hi = w[wide ? 2 * i + 1 : i];
    return wide ? (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo) : (int64_t)lo;
  }
};

template <class By>
__device__ __forceinline__ Request request(const dft_paged_attention_args& a, int b) {
  Request q;
  q.r0 = a.cu_seqlens ? By::i32(a.cu_seqlens + b) : (int64_t)b * a.n_new;
  const int64_t n = a.cu_seqlens ? (int64_t)By::i32(a.cu_seqlens + b + 1) - q.r0 : a.n_new;
  q.status = n < 0 || n > a.n_new || q.r0 < 0 || q.r0 + n > a.rows ? DFT_STATUS_SPAN : 0;
  // a cut request's rows are its first ones: those cut off stand behind them
  // (up to 2^31 - 2^16 of them, as many as rows can be)
  const int given = (int)min(max(n, (int64_t)0), (int64_t)0x7fff0000);
  const int64_t there = q.r0 < 0 ? 0 : max(a.rows - q.r0, (int64_t)0);
  q.n = min(min(given, a.n_new), (int)min(there, (int64_t)0x7fffffff));
  const int64_t top = 0x7fffffff - kTile, room = (int64_t)a.columns * a.page_size;
  const int64_t seq = max(By::index(a.seq_len, b, a.seq_len_dtype), (int64_t)0);
  if (seq > room) q.status |= DFT_STATUS_TABLE;
  q.before = (int)(min(seq, top) - given);
  q.keys = a.num_pages ? (int)min(min(seq, room), top) : 0;
  return q;
}

// Tiles of the row tile's keys; one where it has none, so that its rows are written.
template <int BM, int KT>
__device__ __forceinline__ int tiles_of(const dft_paged_attention_args& a, const Request& q, int group, int tile) {
  int keys = q.keys;
  if (a.flags & DFT_ATTN_CAUSAL) {
    const uint32_t end = (uint32_t)min((tile + 1) * BM, q.n * group);
    keys = min(keys, q.before + (int)((end - 1) / (uint32_t)group) + 1);
  }
  return max((keys + KT - 1) / KT, 1);
}

template <int BM>
__device__ __forceinline__ int row_tiles_of(const Request& q, int group) {
  return (q.n * group + BM - 1) / BM;
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

// One of the rows of an item
struct Place {
  int64_t row;
  int h;
  bool there;
};
__device__ __forceinline__ Place place_of(const Request& q, int group, int g, int p) {
  const int rows = q.n * group, r = min(p, rows - 1);
  const int i = (int)((uint32_t)r / (uint32_t)group);
  return {q.r0 + i, g * group + (r - i * group), p < rows};
}

// A workgroup's walk over its share, from its last item back to its first.  A
// share of a request with many row tiles mostly holds the end of one item and
// the beginning of the next; taken in this order the shares beside it stand at
// the same keys or one same distance further on, and find them in the L2 (two
// chunks of 1024 over 15000: 2.2 GB read past it from first to last, so 0.42;
// 459 us, so 431).
template <int BM, int KT, int NT>
struct Walk {
  int64_t left;  // tiles of the share that are not done
  int g, share;  // kv head, number of the share on its line
  int b, tile;   // the item
  int off, stop, all;  // the share's tiles of it, how many it has
  Request q;

  // An item's tile on the line, found by the thread whose requests hold it.
  struct Found {
    Request q;
    int b, tile, off;
  };
  template <class Weight>
  static __device__ __forceinline__ Found find(const dft_paged_attention_args& a, int group, int b, int64_t rest,
                                               Weight weight) {
    Found f;
    for (int64_t w; rest >= (w = weight(b)); ++b) rest -= w;
    f.q = request<ByLane>(a, b);
    f.b = b;
    f.tile = 0;
    for (int n; rest >= (n = tiles_of<BM, KT>(a, f.q, group, f.tile)); ++f.tile) rest -= n;
    f.off = (int)rest;
    return f;
  }

  __device__ __forceinline__ bool begin(const dft_paged_attention_args& a, const Plan& pl, int group) {
    __shared__ int64_t red[NT / 64];
    __shared__ int at[3];
    if (pl.uncut) {
      const int pairs = a.batch * a.hkv;
      tile = blockIdx.x / pairs;
      const int pair = blockIdx.x - tile * pairs;
      b = pair / a.hkv;
      g = pair - b * a.hkv;
      share = 0;
      off = 0;
      q = request<ByWave>(a, b);
      if (a.status && tile == 0 && g == 0 && threadIdx.x == 0) a.status[b] = q.status;
      if (tile >= row_tiles_of<BM>(q, group)) return false;
      left = stop = all = tiles_of<BM, KT>(a, q, group, tile);
      return true;
    }
    // consecutive shares of a line on one XCD
    const int x = (blockIdx.x % kXcds) * (gridDim.x / kXcds) + blockIdx.x / kXcds;
    g = x / pl.shares;
    share = x - g * pl.shares;
    if (g >= a.hkv) return false;
    const int per = (a.batch + NT - 1) / NT;
    const int b0 = min((int)threadIdx.x * per, a.batch), b1 = min(b0 + per, a.batch);
    auto weight = [&](int r) -> int64_t {
      const Request q = request<ByLane>(a, r);
      if (a.status && x == 0) a.status[r] = q.status;
      int64_t sum = 0;
      const int n = row_tiles_of<BM>(q, group);
      for (int t = 0; t < n; ++t) sum += tiles_of<BM, KT>(a, q, group, t);
      return sum;
    };
    int64_t mine = 0, total;
    for (int r = b0; r < b1; ++r) mine += weight(r);
    const int64_t ahead = scan<NT>(mine, red, total);
    // (a share's tiles in 31 bits: 2^36 keys, some hours' work)
    const int64_t size = max((total + pl.shares - 1) / pl.shares, (int64_t)((BM <= 32 ? kLeastFew : kLeastMany) / KT)), pos = share * size;
    left = min(size, total - pos);
    Head* head = reinterpret_cast<Head*>(pl.heads) + x;
    if (left > 0) {
      const int64_t last = pos + left - 1;
      if (pos >= ahead && pos < ahead + mine) {
        const Found f = find(a, group, b0, pos - ahead, weight);
        Head h;
        h.first = pos - f.off;
        h.last = h.first + tiles_of<BM, KT>(a, f.q, group, f.tile);
        h.share = size;
        h.b = f.b, h.tile = f.tile, h.inside = f.off > 0, h.pad = 0;
        *head = h;
      }
      if (last >= ahead && last < ahead + mine) {
        const Found f = find(a, group, b0, last - ahead, weight);
        at[0] = f.b, at[1] = f.tile, at[2] = f.off;
      }
    } else if (threadIdx.x == 0) {
      head->inside = 0;
    }
    __syncthreads();
    if (left <= 0) return false;
    b = __builtin_amdgcn_readfirstlane(at[0]);
    tile = __builtin_amdgcn_readfirstlane(at[1]);
    stop = __builtin_amdgcn_readfirstlane(at[2]) + 1;
    left = uniform64(left);
    off = (int)max(stop - left, (int64_t)0);
    q = request<ByWave>(a, b);
    all = tiles_of<BM, KT>(a, q, group, tile);
    return true;
  }

  // to the item in front; false past the share's first
  __device__ __forceinline__ bool next(const dft_paged_attention_args& a, int group) {
    left -= stop - off;
    if (left <= 0) return false;
    if (--tile < 0) {
      do {
        if (--b < 0) {
          left = 0;
          return false;
        }
        q = request<ByWave>(a, b);
      } while (q.n == 0);
      tile = row_tiles_of<BM>(q, group) - 1;
    }
    stop = all = tiles_of<BM, KT>(a, q, group, tile);
    off = (int)max(stop - left, (int64_t)0);
    return true;
  }

  template <int D>
  __device__ __forceinline__ float* part(const Plan& pl, bool begins) const {
    return pl.parts + (((int64_t)g * pl.shares + share) * 2 + begins) * part_floats<D, BM>();
  }
};

// Where the value pieces lie: few_kernel reads them by 16 lanes of 4
// consecutive rows each over 2 pieces.
template <int D>
__device__ __forceinline__ int few_value_swizzle(int row) {
  return D == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1;
}

// s_waitcnt: until at most n vector-memory operations are outstanding
constexpr unsigned wait_loads(int n) { return (unsigned)((n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8)); }

// The copies of a share's tiles, item after item, into STAGES places of the
// LDS, STAGES - 1 tiles ahead of their use, and of their keys' page ids, as
// many tiles ahead of the copies.  Every wave fetches the same ids to the same
// place (it then only waits for itself) and copies its share of the rows; a
// wave's loads are the same number for every tile, so that a counted wait ends
// with a tile's.  FEW: the values' places are those of few_value_swizzle.
template <int D, int KT, int NW, int STAGES, bool ONCE, bool FEW, class Walk>
struct Feed {
  // many_kernel forms a tile's scores beside the second product of the tile
  // before it: its keys are fed a tile ahead of its values
  static constexpr int kSkew = FEW ? 0 : 1;
  static constexpr int kRow = 2 * D, kBytes = KT * kRow, kAhead = STAGES - 1, kSlots = STAGES > 2 ? 8 : 4;
  static constexpr int kRows = 1024 / kRow, kCopies = KT / (kRows * NW), kPieces = D / 8, kLoads = 2 * kCopies + 1;
  static constexpr int kMine = kCopies * kRows;  // rows of a tile that a wave copies
  struct Room {
    char keys[STAGES][kBytes], values[STAGES][kBytes];
    uint64_t from[NW][2 * kMine];  // addresses of a wave's keys of a tile, and of its values
    int ids[kSlots][64];           // page ids of a tile's keys; with 32 of them twice
    int2 tile[kSlots];             // its first key and its item's number of keys
  };

  const dft_paged_attention_args& a;
  const Plan& pl;
  Room& room;
  Walk lead;  // the walk as far as the ids
  int ahead;  // and its tile of the item
  int group;
  uint64_t id_at;        // the last ids fetched
  int id_slot;
  int ids, count, used;  // tiles whose ids are fetched; of the share; behind us
  uint64_t base;         // of what the lane looks up: keys or values
  int64_t page_stride, token_stride;
  int wave, lane;

  __device__ __forceinline__ Feed(const dft_paged_attention_args& a, const Plan& pl, Room& room, const Walk& walk, int group,
                                  int wave)
      : a(a), pl(pl), room(room), lead(walk), ahead(walk.off), group(group), id_at(0), id_slot(0), ids(0), count((int)walk.left), used(0),
        wave(wave), lane(threadIdx.x & 63) {
    const bool value = lane & kMine;
    base = value ? (uint64_t)(uintptr_t)a.value_cache + 2 * (walk.g * a.vc_h_stride)
                 : (uint64_t)(uintptr_t)a.key_cache + 2 * (walk.g * a.kc_h_stride);
    page_stride = value ? a.vc_page_stride : a.kc_page_stride;
    token_stride = value ? a.vc_token_stride : a.kc_token_stride;
  }
  // where the keys and the values of tile n are
  __device__ __forceinline__ uint32_t keys_at(int n) const {
    return lds_address(room.keys) + (n & (STAGES - 1)) * kBytes;
  }
  __device__ __forceinline__ uint32_t values_at(int n) const {
    return lds_address(room.values) + (n & (STAGES - 1)) * kBytes;
  }
  __device__ __forceinline__ uint32_t column(uint32_t j) const { return (uint32_t)((uint64_t)j * pl.magic >> pl.shift); }

  // the next tile's ids; past the share's end the last ones again, for the count
  __device__ __forceinline__ void fetch_ids() {
    if (ids < count) {
      id_slot = ids & (kSlots - 1);
      const int j0 = ahead * KT;
      const uint32_t j = (uint32_t)max(min(j0 + lane % KT, lead.q.keys - 1), 0);
      id_at = (uint64_t)(uintptr_t)(a.block_table + lead.b * a.table_row_stride + column(j));
      room.tile[id_slot] = int2{j0, lead.q.keys};
      ++ids;
      if (++ahead == lead.stop) {
        lead.next(a, group);
        ahead = lead.off;
      }
    }
    dma4_at(id_at, lds_address(room.ids[id_slot]));
  }
  // -1 for a key that there is, 0 for none.  Arithmetic, as what follows in
  // copy(): a branch of some lanes only among so many live registers let the
  // compiler put register copies in front of the rejoin, where they left out
  // the other lanes (a memory fault at 256 columns in fp16).
  __device__ __forceinline__ int there(int j, int keys, int id) const {
    return -(int)((j < keys) & ((uint32_t)id < (uint32_t)a.num_pages));
  }
  // The values of tile n and the keys of tile n + kSkew (past the share's end
  // the last tile's again), in parts that many_kernel spreads over its
  // products: look up, place, send the keys, send the values.
  int looked_j, looked_id, looked_keys;  // of the row that the lane looks up, for the keys or for the values
  __device__ __forceinline__ void look_up(int n) {
    const int of_keys = min(n + kSkew, count - 1);
    const int slot = (lane & kMine ? n : of_keys) & (kSlots - 1), mine = lane % kMine;
    const int row = (mine / kRows * NW + wave) * kRows + mine % kRows;
    const int2 tile = room.tile[slot];
    looked_j = tile.x + row;
    looked_keys = tile.y;
    looked_id = room.ids[slot][row];
  }
  __device__ __forceinline__ void place() {
    const int j = looked_j, ok = there(j, looked_keys, looked_id);
    const uint64_t page = (uint32_t)(looked_id & ok), token = (j - column(j) * a.page_size) & ok;
    room.from[wave][lane & (2 * kMine - 1)] = base + 2 * (page * page_stride + token * token_stride);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
  __device__ __forceinline__ void send(int n, bool values) {
    uint64_t at[kCopies];
#pragma unroll
    for (int x = 0; x < kCopies; ++x) {
      const int to = (x * NW + wave) * kRows + lane / kPieces, piece = lane % kPieces;
      const int swizzle = !values ? key_swizzle<D>(to) : FEW ? few_value_swizzle<D>(to) : value_swizzle<D>(to);
      at[x] = room.from[wave][x * kRows + lane / kPieces + (values ? kMine : 0)] + ((piece ^ swizzle) << 4);
    }
    dma16_at<kCopies, 1024 * NW, ONCE>(at, (values ? values_at(n) : keys_at(n + kSkew)) + 1024 * wave);
  }
  __device__ __forceinline__ void copy(int n) {
    look_up(n);
    place();
    send(n, false);
    send(n, true);
  }
  // which of tile n's keys, from j0 on, there are
  __device__ __forceinline__ uint64_t present(int n, int j0, int keys) const {
    return __ballot(there(j0 + lane % KT, keys, room.ids[n & (kSlots - 1)][lane]));
  }

  // the share's first tiles
  __device__ __forceinline__ void begin() {
#pragma unroll 1
    for (int t = 0; t < 2 * kAhead + kSkew; ++t) fetch_ids();
    __builtin_amdgcn_s_waitcnt(kWaitDma);
    asm volatile("" ::: "memory");
    if constexpr (kSkew) {
      look_up(-1);
      place();
      send(-1, false);
    }
#pragma unroll 1
    for (int t = 0; t < min(kAhead, count); ++t) {
      dma4_at(id_at, lds_address(room.ids[id_slot]));
      copy(t);
    }
    if constexpr (kSkew) {  // the first tile's keys, for all waves
      wait(1);
      __syncthreads();
    }
  }
  // until this wave's copies are done, but for those of `behind` tiles
  __device__ __forceinline__ void wait(int behind) const {
    static_assert(kAhead == (FEW ? 3 : 1));  // behind: at most 2, or 1
    if (FEW && behind == 2)
      __builtin_amdgcn_s_waitcnt(wait_loads(2 * kLoads));
    else if (behind == 1)
      __builtin_amdgcn_s_waitcnt(wait_loads(kLoads));
    else
      __builtin_amdgcn_s_waitcnt(kWaitDma);
  }
  // the current tile, for all waves
  __device__ __forceinline__ void ready() {
    wait(min(count - 1 - used, kAhead - 1));
    __syncthreads();
  }
  // sends for the tile kAhead from here
  __device__ __forceinline__ void advance() {
    if (used + kAhead >= count) return;
    fetch_ids();
    copy(used + kAhead);
  }
  // the same in parts, 0 .. 3
  __device__ __forceinline__ void advance(int part) {
    if (used + kAhead >= count) return;
    if (part == 0) {
      fetch_ids();
      look_up(used + kAhead);
    } else if (part == 1) {
      place();
    } else {
      send(used + kAhead, part == 3);
    }
  }
};

// A tree row's visible keys of the 64 from j0 on.
__device__ __forceinline__ uint64_t tree_bits(uint64_t bits, int before, int j0) {
  const int up = before - j0;
  return first_bits(up) | (up >= 64 || up <= -64 ? 0 : up >= 0 ? bits << up : bits >> -up);
}

// ---- up to 32 rows ---------------------------------------------------------
// All four waves work on the same 32-key tiles: each forms the scores of all
// rows (on 16 x 16 products, half the work of 32 x 32 ones for the 4 to 16
// rows of a decode step) and takes a quarter of the output's columns, so
// nothing is exchanged between them.  Four tiles' room in the LDS keeps three
// on their way, 72 to 96 KB a CU: bound by HBM, and HBM by what is on its way.
// 64 requests of 300 to 8191 keys (8 kv heads, d 128): 184 us, 6.0 TB/s; two
// waves on halves of 64-key tiles two deep took 249, copies without the
// read-once mark 218.
constexpr int kFewTile = 32, kFewStages = 4;

// V^T fragment: 16 columns, the tile's 32 keys in the order of the weights
template <int D, class T>
__device__ __forceinline__ typename T::x8 few_value(uint32_t v, int columns) {
  const int lane = threadIdx.x & 63, row = 4 * (lane >> 4) + ((lane & 15) >> 2);
  const uint32_t at = v + row * 2 * D + (((((lane & 3) >> 1) ^ few_value_swizzle<D>(row)) << 4) ^ (columns << 5)) + ((lane & 1) << 3);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DFT_LDS s16x4*)(uintptr_t)at);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DFT_LDS s16x4*)(uintptr_t)(at + 16 * 2 * D));
  return __builtin_bit_cast(typename T::x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// One tile for NQ x 16 rows (lane l: row l % 16) and the wave's DT x 16
// columns.  As Rows::scores and Rows::step, on 16 x 16 products.
template <int D, int NQ, int DT, class T>
__device__ __forceinline__ void few_tile(uint32_t k, uint32_t v, int wave, const typename T::x8 (&q)[NQ][D / 32],
                                         f32x4 (&o)[NQ][DT], float (&top)[NQ], float (&sum)[NQ], float c, bool partial,
                                         const uint32_t (&vis)[NQ]) {
  typedef typename T::x8 x8;
  const int lane = threadIdx.x & 63, quad = lane >> 4, row = lane & 15;
  const uint32_t ka = k + row * 2 * D + ((quad ^ key_swizzle<D>(row)) << 4);
  f32x4 s[NQ][2];
#pragma unroll
  for (int y = 0; y < NQ; ++y) s[y][0] = s[y][1] = f32x4{};
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const x8 kf = *(const DFT_LDS x8*)(uintptr_t)((ka ^ (j << 6)) + t * 16 * 2 * D);
#pragma unroll
      for (int y = 0; y < NQ; ++y) s[y][t] = T::mfma16(kf, q[y][j], s[y][t]);
    }
  x8 p[NQ];
#pragma unroll
  for (int y = 0; y < NQ; ++y) {
    if (partial) {
      const uint32_t mine = vis[y] >> (4 * quad);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[y][t][r] = __uint_as_float(select(__float_as_uint(s[y][t][r]), 0xff800000u, mine, 16 * t + r));
    }
    float high = s[y][0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) high = fmaxf(high, s[y][t][r]);
    constexpr float kMost = T::kBase + T::kSlack;
    if (__any(high * c > top[y] + kMost)) {
      high = fmaxf(high, __shfl_xor(high, 16));
      const float new_top = fmaxf(high, __shfl_xor(high, 32)) * c;
      const bool move = new_top - top[y] > kMost;
      const float next = move ? new_top - T::kBase : top[y], by = move ? __builtin_amdgcn_exp2f(top[y] - next) : 1.f;
      top[y] = next;
      sum[y] *= by;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[y][d] *= by;
    }
    const float sub = top[y] == -INFINITY ? 0.f : top[y];
    f32x8 e;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      e[x] = __builtin_amdgcn_exp2f(fmaf(s[y][x / 4][x % 4], c, -sub));
      sum[y] += e[x];
    }
    p[y] = __builtin_convertvector(e, x8);
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const x8 vf = few_value<D, T>(v, wave * DT + d);
#pragma unroll
    for (int y = 0; y < NQ; ++y) o[y][d] = T::mfma16(vf, p[y], o[y][d]);
  }
}

// As Rows::note: 2 words a lane and row block, 4 bits a column block.
template <int D, int NQ, int DT, class T>
__device__ __forceinline__ void note_few(uint32_t v, int wave, const uint32_t (&vis)[NQ], uint32_t notes, bool noted) {
  typedef typename T::x8 x8;
  const int lane = threadIdx.x & 63;
  DFT_LDS uint32_t* note = (DFT_LDS uint32_t*)(uintptr_t)(notes + 4 * lane);
#pragma unroll
  for (int y = 0; y < NQ; ++y) {
    const uint32_t mine = vis[y] >> (4 * (lane >> 4));
    u32x4 seen;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t bits = mine >> (16 * (x / 2) + 2 * (x % 2));
      seen[x] = (bits & 1) * T::kOne + (bits >> 1 & 1) * (T::kOne << 16);
    }
#pragma unroll
    for (int sign = 0; sign < 2; ++sign) {
      uint32_t word = noted ? note[64 * (2 * y + sign)] : 0;
#pragma unroll 1
      for (int d = 0; d < DT; ++d) {
        const u32x4 w = __builtin_bit_cast(u32x4, few_value<D, T>(v, wave * DT + d));
        u32x4 flag;
#pragma unroll
        for (int x = 0; x < 4; ++x) flag[x] = infinite<T>(w[x], sign) + (infinite<T>(w[x] >> 16, sign) << 16);
        const f32x4 n = T::mfma16(__builtin_bit_cast(x8, flag), __builtin_bit_cast(x8, seen), f32x4{});
#pragma unroll
        for (int r = 0; r < 4; ++r) word |= min(__float_as_uint(n[r]), 1u) << (4 * d + r);
      }
      note[64 * (2 * y + sign)] = word;
    }
  }
}

template <int D, int NQ, class T>
__global__ void __launch_bounds__(256) few_kernel(dft_paged_attention_args a, Scale sc, Plan pl) {
  constexpr int BM = 16 * NQ, KT = kFewTile, NW = 4, QK = D / 32, DT = D / 16 / NW;
  typedef Walk<BM, KT, 64 * NW> Share;
  typedef Feed<D, KT, NW, kFewStages, true, true, Share> Tiles;
  typedef typename T::x8 x8;
  __shared__ __attribute__((aligned(1024))) typename Tiles::Room room;
  __shared__ uint32_t notes[NW][NQ * 2][64];
  __shared__ int spoiled;  // the last tile found to hold a value that is not finite
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4;
  const int group = a.hq / a.hkv;
  const bool causal = a.flags & DFT_ATTN_CAUSAL;
  Share walk;
  if (!walk.begin(a, pl, group)) return;
  Tiles feed(a, pl, room, walk, group, wave);
  if (threadIdx.x == 0) spoiled = -1;
  feed.begin();

  bool more = true;
  while (more) {
    const Request q = walk.q;
    const int begin = walk.off, stop = walk.stop;
    Place to[NQ];
    uint64_t bits[NQ];
    int limit[NQ], fewest = q.keys;
#pragma unroll
    for (int y = 0; y < NQ; ++y) {
      to[y] = place_of(q, group, walk.g, walk.tile * BM + 16 * y + (lane & 15));
      limit[y] = q.keys;
      bits[y] = a.anc_bits ? a.anc_bits[to[y].row] : 0;
      if (causal) limit[y] = min(q.before + (int)(to[y].row - q.r0) + 1, q.keys);
    }
    if (a.anc_bits)
      fewest = q.before;
    else if (causal)
      fewest = __builtin_amdgcn_readlane(limit[0], 0);

    x8 qf[NQ][QK];
    f32x4 o[NQ][DT];
    float top[NQ], sum[NQ];
    bool noted = false;
#pragma unroll
    for (int y = 0; y < NQ; ++y) {
      top[y] = -INFINITY;
      sum[y] = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[y][d] = f32x4{};
    }
#pragma unroll
    for (int y = 0; y < NQ; ++y) {
      const uint16_t* row = static_cast<const uint16_t*>(a.q) + to[y].row * a.q_row_stride + to[y].h * a.q_h_stride;
#pragma unroll
      for (int k = 0; k < QK; ++k) {
        u32x4 w = *reinterpret_cast<const u32x4*>(row + 32 * k + 8 * quad);
        w = (w & sc.keep) ^ sc.flip;
        qf[y][k] = __builtin_bit_cast(x8, w);
      }
    }
    for (int t = begin; t < stop; ++t, ++feed.used) {
      feed.ready();
      feed.advance();
      const uint32_t kt = feed.keys_at(feed.used), vt = feed.values_at(feed.used);
      const int j0 = t * KT;
      const uint32_t there = (uint32_t)feed.present(feed.used, j0, q.keys);
      const bool partial = there != ~0u || j0 + KT > fewest;
      uint32_t vis[NQ];
      if (partial) {
#pragma unroll
        for (int y = 0; y < NQ; ++y)
          vis[y] = there & (uint32_t)(a.anc_bits ? tree_bits(bits[y], q.before, j0) : first_bits(limit[y] - j0));
        const uint32_t slice = vt + wave * (Tiles::kBytes / NW);
        if (!finite<T, Tiles::kBytes / NW>(slice)) spoiled = feed.used;
        __syncthreads();
        if (spoiled == feed.used) {
          note_few<D, NQ, DT, T>(vt, wave, vis, lds_address(notes[wave]), noted);
          noted = true;
          __syncthreads();
          clear_infinite<T, Tiles::kBytes / NW>(slice);
          __syncthreads();
        }
      }
      few_tile<D, NQ, DT, T>(kt, vt, wave, qf, o, top, sum, sc.c, partial, vis);
    }

    const bool whole = begin == 0 && stop == walk.all;
    float* part = walk.template part<D>(pl, begin == 0);
#pragma unroll
    for (int y = 0; y < NQ; ++y) {
      sum[y] += __shfl_xor(sum[y], 16);
      sum[y] += __shfl_xor(sum[y], 32);
      const float by = whole ? weight_of(sum[y]) : 1.f;
      if (noted) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint32_t up = notes[wave][2 * y][lane] >> (4 * d), down = notes[wave][2 * y + 1][lane] >> (4 * d);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            o[y][d][r] += __uint_as_float(select(0x7f800000u, 0, up, r));
            o[y][d][r] += __uint_as_float(select(0xff800000u, 0, down, r));
          }
        }
      }
      if (!to[y].there) continue;
      if (whole)
        store_all<DT>(a.o, to[y].row * a.o_row_stride + to[y].h * a.o_h_stride + 16 * wave * DT + 4 * quad, a.o_dtype, pl.vec,
                      [&](int d) { return o[y][d] * by; }, [](int d) { return 16 * d; });
      else
#pragma unroll
        for (int d = 0; d < DT; ++d)
          *reinterpret_cast<f32x4*>(part + ((y * (D / 16) + wave * DT + d) * 64 + lane) * 4) = o[y][d];
      if (wave || quad) continue;
      if (!whole) {
        part[BM * D + 16 * y + lane] = top[y];
        part[BM * D + BM + 16 * y + lane] = sum[y];
      } else if (a.lse) {
        a.lse[to[y].row * a.lse_row_stride + to[y].h] = lse_of(top[y], sum[y]);
      }
    }
    more = walk.next(a, group);
  }
}

// ---- more rows -------------------------------------------------------------
// NW waves of 32 rows each, on 64-key tiles two deep: 32-key tiles four deep
// cost more per tile than their deeper pipeline gives (draft trees 156 us for
// 148, chunks 740 for 516 on one build).  With 128 columns two workgroups
// share a CU; with 256 the accumulators leave room for one wave a SIMD, whose
// products and everything else then overlap within the wave only.  32-node
// trees of 64 requests over 500 to 4000 keys (8 kv heads, d 128): 148 us,
// 4.3 TB/s and 510 TFLOP/s, 16 more for the join; chunks of 777 and 1024 rows
// over 9000 to 15001 keys (2 kv heads, d 256): 430 us with the join's 16, 820
// TFLOP/s (the profiler makes it 444 to 462 and 16).  Some 50 of them pass
// before the first key: one thread walks a request's row tiles (Walk::begin),
// which takes 500 us of a chunk of 16384 tokens, 8 heads each, out of 3880.
template <int D, int NW, int KT, int STAGES, bool ONCE, class T>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) many_kernel(dft_paged_attention_args a, Scale sc, Plan pl) {
  constexpr int BM = 32 * NW;
  typedef Walk<BM, KT, 64 * NW> Share;
  typedef Feed<D, KT, NW, STAGES, ONCE, false, Share> Tiles;
  typedef Rows<D, KT, T> Wave;
  constexpr int kBytes = Tiles::kBytes;
  constexpr uint64_t kEvery = KT == 64 ? ~0ull : (1ull << KT) - 1;
  __shared__ __attribute__((aligned(1024))) typename Tiles::Room room;
  __shared__ char notes[NW][Wave::kNotes];
  __shared__ int spoiled;  // the last tile found to hold a value that is not finite
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int group = a.hq / a.hkv;
  const bool causal = a.flags & DFT_ATTN_CAUSAL;
  Share walk;
  if (!walk.begin(a, pl, group)) return;
  Tiles feed(a, pl, room, walk, group, wave);
  if (threadIdx.x == 0) spoiled = -1;
  feed.begin();
  Wave w;
  w.notes = lds_address(notes[wave]);

  bool more = true;
  while (more) {
    const Request q = walk.q;
    const int begin = walk.off, stop = walk.stop;
    const int rows = q.n * group, pw = walk.tile * BM + 32 * wave;
    const bool works = pw < rows;
    const Place to = place_of(q, group, walk.g, pw + (lane & 31));
    const int fewest = a.anc_bits ? q.before  // keys that every row of the workgroup sees
                       : causal   ? min(q.before + (int)((uint32_t)(walk.tile * BM) / (uint32_t)group) + 1, q.keys)
                                  : q.keys;
    uint64_t bits = 0;
    int limit = q.keys, least = q.keys;  // keys the lane's row sees, all rows of the wave do
    if (a.anc_bits) {
      bits = a.anc_bits[to.row];
      least = q.before;
    } else if (causal) {
      limit = min(q.before + (int)(to.row - q.r0) + 1, q.keys);
      least = __builtin_amdgcn_readlane(limit, 0);
    }

    w.clear();
    w.load_q(static_cast<const uint16_t*>(a.q) + to.row * a.q_row_stride + to.h * a.q_h_stride, sc);
    // the keys there are of the tile at hand, from j0 on, and of the next one
    int j0 = begin * KT;
    uint64_t there = feed.present(feed.used, j0, q.keys) & kEvery;
    auto seen = [&](uint64_t here, int from) {
      return here & (a.anc_bits ? tree_bits(bits, q.before, from) : first_bits(limit - from));
    };
    typename Wave::Scores s;
    w.scores(feed.keys_at(feed.used), s);
    if (there != kEvery || j0 + KT > least) w.mask(s, seen(there, j0));
    // what of a tile's values is not finite must not reach a row that does not see it
    auto look = [&](uint32_t vt) {
      if (there == kEvery && j0 + KT <= fewest) return;
      const uint32_t slice = vt + wave * (kBytes / NW);
      if (!finite<T, kBytes / NW>(slice)) spoiled = feed.used;
      __syncthreads();
      if (spoiled == feed.used) {
        w.note(vt, seen(there, j0));
        __syncthreads();
        clear_infinite<T, kBytes / NW>(slice);
        __syncthreads();
      }
    };
    for (int t = begin; t + 1 < stop; ++t) {
      feed.ready();
      look(feed.values_at(feed.used));
      w.template step<true>(feed.keys_at(feed.used + 1), feed.values_at(feed.used), sc.c, s,
                            [&](int part) { feed.advance(part); });
      ++feed.used;
      j0 += KT;
      there = feed.present(feed.used, j0, q.keys) & kEvery;
      if (there != kEvery || j0 + KT > least) w.mask(s, seen(there, j0));
    }
    feed.ready();
    look(feed.values_at(feed.used));
    w.template step<false>(0, feed.values_at(feed.used), sc.c, s, [&](int part) { feed.advance(part); });
    ++feed.used;
    w.finish();

    if (works) {
      const bool whole = begin == 0 && stop == walk.all;
      const float sum = w.whole_sum(), by = weight_of(sum);
      if (to.there) {
        float* part = walk.template part<D>(pl, begin == 0);
        if (whole) {
          w.store(a.o, to.row * a.o_row_stride + to.h * a.o_h_stride, a.o_dtype, pl.vec, by);
        } else {
#pragma unroll
          for (int t = 0; t < Wave::DT; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              *reinterpret_cast<f32x4*>(part + (((wave * Wave::DT + t) * 4 + x) * 64 + lane) * 4) = w.four(t, x);
        }
        if (half == 0) {
          if (!whole) {
            part[BM * D + 32 * wave + lane] = w.top;
            part[BM * D + BM + 32 * wave + lane] = sum;
          } else if (a.lse) {
            a.lse[to.row * a.lse_row_stride + to.h] = lse_of(w.top, sum);
          }
        }
      }
    }
    more = walk.next(a, group);
  }
}

// ---- the join --------------------------------------------------------------
// Joins the parts of the items that share boundaries cut.  The workgroups of
// an item's boundaries deal its units out among them: as many workgroups as
// there are parts to read, times four with many rows, whose parts have four
// times a workgroup's units (5 to 6 us at 16 rows an item; at 128 rows 10 for
// four trees, 15.6 for 64, where it moves 100 MB, 16.5 in both with one each;
// a workgroup per part and unit, most of them idle, took 13 and 31).  With few parts a wave takes a unit, with many the
// waves divide a unit's parts.
constexpr int kJoinWaves = 8;

template <int D, int BM>
__global__ void __launch_bounds__(64 * kJoinWaves) join_kernel(dft_paged_attention_args a, Plan pl) {
  // rows of a block of units, units of it, of all
  constexpr int kLane = BM <= 32 ? 16 : 32, kOf = kLane == 16 ? D / 16 : D / 8, kUnits = BM / kLane * kOf;
  const int x = blockIdx.x, g = x / pl.shares, share = x - g * pl.shares;
  const Head h = reinterpret_cast<const Head*>(pl.heads)[x];
  if (!h.inside) return;
  __shared__ f32x4 sums[kJoinWaves][64];
  __shared__ float tops[kJoinWaves][64], totals[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = a.hq / a.hkv;
  const int64_t begin = h.first / h.share, past = (h.last - 1) / h.share;  // the item's first and last share
  const int parts = (int)(past - begin) + 1, split = parts > 8 ? kJoinWaves : 1;
  const int units = kJoinWaves / split, turn = wave % split;  // units at a time; which of the parts
  const float* first = pl.parts + ((int64_t)g * pl.shares + begin) * 2 * part_floats<D, BM>();
  const Request q = request<ByWave>(a, h.b);
  const int step = (parts - 1) * (int)gridDim.y * units;
  for (int u0 = ((share - 1 - (int)begin) * (int)gridDim.y + blockIdx.y) * units; u0 < kUnits; u0 += step) {
    const int unit = min(u0 + wave / split, kUnits - 1), block = unit / kOf, in = unit % kOf;
    const int row = block * kLane + lane % kLane;
    const int d = kLane == 16 ? 16 * in + 4 * (lane / 16) : 8 * in + 4 * (lane / 32);
    const Place to = place_of(q, group, g, h.tile * BM + row);
    float top = -INFINITY, sum = 0;
    f32x4 o = {};
    if (to.there) {
#pragma unroll 4
      for (int s = turn; s < parts; s += split) {
        const float* part = first + (int64_t)(2 * s + (s == 0)) * part_floats<D, BM>();
        const float his = part[BM * D + row], high = fmaxf(top, his), add = part[BM * D + BM + row];
        const f32x4 y = *reinterpret_cast<const f32x4*>(part + (unit * 64 + lane) * 4);
        const float by = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - high);
        const float with = his == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(his - high);
        top = high;
        sum = sum * by + add * with;
        o = o * by + y * with;
      }
    }
    if (split > 1) {
      tops[wave][lane] = top;
      totals[wave][lane] = sum;
      sums[wave][lane] = o;
      __syncthreads();
#pragma unroll
      for (int s = 0; s < kJoinWaves; ++s) top = fmaxf(top, tops[s][lane]);
      sum = 0;
      o = f32x4{};
#pragma unroll
      for (int s = 0; s < kJoinWaves; ++s) {
        const float his = tops[s][lane], by = his == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(his - top);
        sum += totals[s][lane] * by;
        o += sums[s][lane] * by;
      }
      __syncthreads();
    }
    if (turn || !to.there || u0 + wave / split >= kUnits) continue;
    store_all<1>(a.o, to.row * a.o_row_stride + to.h * a.o_h_stride + d, a.o_dtype, pl.vec,
                 [&](int) { return o * weight_of(sum); }, [](int) { return 0; });
    if (a.lse && d == 0) a.lse[to.row * a.lse_row_stride + to.h] = lse_of(top, sum);
  }
}

// The status words of a launch without rows.
__global__ void __launch_bounds__(256) status_kernel(dft_paged_attention_args a) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.batch) a.status[b] = request<ByLane>(a, b).status;
}

// The launch's sizes.
struct Shape {
  int rows;  // of an item: 16, 32 (few_kernel), 128 (many_kernel)
  bool once, uncut;
  int64_t grid, shares, heads_bytes, parts_bytes;
};
Shape shape_of(const dft_paged_attention_args& a) {
  Shape s = {};
  const int64_t rows = (int64_t)a.n_new * (a.hq / a.hkv);
  // trees of 4 and 8 nodes (16 and 32 rows, 64 requests over 500 to 4000 keys):
  // 138 and 142 us with few_kernel, 158 and 152 with many_kernel
  s.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 128;
  s.once = rows <= s.rows;  // a key is read for one item only
  // a grid counts work-items, 256 a workgroup, in 32 bits: a large n_new over a
  // large batch can ask for more, most of them for rows that there are not
  s.grid = (int64_t)a.batch * a.hkv * ((rows + s.rows - 1) / s.rows);
  s.uncut = (int64_t)a.columns * a.page_size <= kUncutKeys && s.grid <= 0xffffffffll / 256;
  if (s.uncut) return s;
  // As many workgroups as a CU takes at once with 256 and 128 columns, whose
  // tiles are 512 D bytes of the LDS each.  With 64 columns three, between two
  // (as many as many_kernel's registers allow) and four (as the LDS does), for
  // a token of 64 requests 137 us (153 and 128), one of 60000 keys 40 (45 and
  // 45), 32-node trees 138 (115 and 131), 8-node ones 99 (102 and 108).
  const int room = kCus * (a.head_dim == 256 ? 1 : a.head_dim == 128 ? 2 : 3);
  s.shares = a.hkv < room ? room / a.hkv : 1;
  s.grid = (s.shares * a.hkv + kXcds - 1) / kXcds * kXcds;
  s.heads_bytes = s.grid * sizeof(Head);
  s.parts_bytes = s.shares * a.hkv * 2 * s.rows * (a.head_dim + 2) * sizeof(float);
  return s;
}

template <int D, class T>
int launch(const dft_paged_attention_args& a, const Shape& s, const Plan& pl, hipStream_t stream) {
  const Scale sc = split_scale(a.scale);
  const unsigned grid = (unsigned)s.grid, lines = (unsigned)(s.shares * a.hkv);
  if (s.rows == 16)
    few_kernel<D, 1, T><<<grid, 256, 0, stream>>>(a, sc, pl);
  else if (s.rows == 32)
    few_kernel<D, 2, T><<<grid, 256, 0, stream>>>(a, sc, pl);
  else if (s.once)
    many_kernel<D, 4, 64, 2, true, T><<<grid, 256, 0, stream>>>(a, sc, pl);
  else
    many_kernel<D, 4, 64, 2, false, T><<<grid, 256, 0, stream>>>(a, sc, pl);
  if (hipGetLastError() != hipSuccess) return DFT_ERR_LAUNCH;
  if (s.uncut) return DFT_OK;
  if (s.rows == 16)
    join_kernel<D, 16><<<lines, 64 * kJoinWaves, 0, stream>>>(a, pl);
  else if (s.rows == 32)
    join_kernel<D, 32><<<lines, 64 * kJoinWaves, 0, stream>>>(a, pl);
  else
    join_kernel<D, 128><<<dim3(lines, 4), 64 * kJoinWaves, 0, stream>>>(a, pl);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

template <class T>
int launch_type(const dft_paged_attention_args& a, const Shape& s, const Plan& pl, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch<64, T>(a, s, pl, stream);
    case 128: return launch<128, T>(a, s, pl, stream);
    default: return launch<256, T>(a, s, pl, stream);
  }
}

}  // namespace

int64_t paged_attention_workspace(const dft_paged_attention_args* a) {
  const Shape s = shape_of(*a);
  return s.heads_bytes + s.parts_bytes;
}

int launch_paged_status(const dft_paged_attention_args* a, hipStream_t stream) {
  status_kernel<<<(a->batch + 255) / 256, 256, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

int launch_paged_attention(const dft_paged_attention_args* args, hipStream_t stream) {
  dft_paged_attention_args copy = *args, *a = &copy;
  // requests without keys pass through the tiles as well, all masked: where
  // there is no table or no page they read something that is there
  if (!a->columns) a->block_table = static_cast<const int32_t*>(a->q), a->table_row_stride = 0;
  if (!a->num_pages) {
    a->key_cache = a->value_cache = a->q;
    a->kc_page_stride = a->kc_token_stride = a->kc_h_stride = a->vc_page_stride = a->vc_token_stride = a->vc_h_stride = 0;
  }
  const Shape s = shape_of(*a);
  Plan pl = {};
  pl.heads = static_cast<char*>(a->workspace);
  pl.parts = reinterpret_cast<float*>(pl.heads + s.heads_bytes);
  page_magic(a->page_size, pl.magic, pl.shift);
  pl.shares = (int)s.shares;
  pl.vec = vector_out(*a);
  pl.uncut = s.uncut;
  return a->dtype == DFT_BF16 ? launch_type<Bf16>(*a, s, pl, stream) : launch_type<F16>(*a, s, pl, stream);
}

}  // namespace dft
