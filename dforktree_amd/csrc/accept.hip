// dft_tree_accept: which drafted tokens stand, and the token behind them.
//
// The walk from the root needs of every node only two values, p and q at its
// token in its parent's rows, which are fetched for all nodes at once; the walk
// itself is a wave's work on them.  What takes time is whole rows: the sum of
// max(r - q, 0) where a refused child has another sibling, and r's running sum
// at the end.  Such a pass over a row is cut into slices, a workgroup each.  A
// launch does one pass for every request, whatever it is of that request's; the
// next one walks again, with the sums there are, to the next pass, until a walk's
// last.  Without the drafter's probabilities the first pass is the last; with
// them up to kRounds launches are made, and what is still open is done by the
// request's workgroup alone in the last launch, which finds the token from the
// sums of its slice: a slice's tokens side by side, added up over the workgroup.
//
// Bound by launches and by the walk's dependent fetches where passes are few: 17
// to 22 us for one request of 16 nodes over 131072 tokens, 31 for 64 drawn chains,
// 20 for 64 trees of 32 nodes without a drafter's rows; of these the last launch
// is 5 to 9, and a launch that finds nothing to do costs 1.4 to 3.  48 drawn trees
// of 8 to 40 nodes over 100003 tokens take 39 to 70, by how many children their
// random numbers refuse.  Their passes are bound by the 64-bit units: a reduction
// divides by two numbers that are the same for the whole row, so it multiplies by
// their reciprocals.
// The passes of a request past the fourth are its one workgroup's, and every pass
// repeats the reductions in front of it: a node over 131072 tokens with 5, 7, 15,
// 39 and 63 refused children takes 99 us, 223 us, 1.0, 6.0 and 15 ms.
//
// Sums are held in 64 bits: a sum of 10^5 probabilities in 32 bits moves one
// drawn token in some hundred over a border.  They are added up in one order.
#include <algorithm>

#include "packed.h"

namespace dft {
namespace {

constexpr int kNodes = 64, kSlices = 64, kRounds = 4, kShort = 16384;
constexpr int kPass = 256, kLast = 512, kWaves = kLast / 64;  // threads of a pass and of the last launch

template <class T>
__device__ __forceinline__ double weight(const void* p, int64_t at, int dt) {
  float x;
  if constexpr (sizeof(T) == 1)
    x = ld_f(p, at, dt);  // any type
  else
    x = (float)static_cast<const T*>(p)[at];
  return x > 0 ? (double)x : 0.0;  // NaN too
}

// What was refused at a node: r is the target's distribution reduced `count`
// times, or with the refused tokens left out where there is no drafter's.
struct Refused {
  int count;
  int token[kNodes];
  // 1 over 1 less the drafter's mass of the tokens in front of this one, and over the sum of the weights left behind it; 0
  // for what counts as none
  double by_off[kNodes], by_sum[kNodes];
};

__device__ __forceinline__ double wave_sum(double x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ int wave_max(int x) {
  for (int o = 32; o; o >>= 1) x = max(x, __shfl_xor(x, o));
  return x;
}

struct Work {
  double* sums;        // [round][batch][kSlices]
  int* tops;           // the same: the last token of any weight, -1 for none
  int* done;           // [round][batch] whether the walk's last pass is made by then
  struct Walk* walks;  // [batch] of those whose is
  int slices, length;  // of a pass; tokens of a slice
};

// A request's walk as far as it goes, in the LDS.
struct Walk {
  Refused f;
  int path[kNodes];
  int node, length, pass;  // where the path stands, its nodes, the pass that comes next
  bool open, last;         // whether that is of the last refusal, and the walk's last
};

// Lane c's value, c the same for all.
__device__ __forceinline__ double of_lane(double x, int c) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)bits, c), hi = __builtin_amdgcn_readlane((uint32_t)(bits >> 32), c);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The walk, by one wave, a node a lane: every lane holds what is left of r and q
// at its own token, so that a refusal costs the same however many there were.
template <bool DRAFT, class T>
struct Walker {
  int parent = -1, token = 0;
  double u = 0, p = 0, q = 0;
  // at the node where the path stands: r at the lane's token, before and after it is divided by the sum, and whether the
  // token has been refused
  double r, rest = 0;
  bool gone = false;
  int node = 0, length, count = 0, pass = 0;
  bool open = false, waits = false;  // (every lane keeps the same of these)
  double off = 0;
  uint64_t kids;

  __device__ __forceinline__ Walker(const dft_tree_accept_args& a, const packed::Span& s, Walk& w) : length(s.n > 0) {
    const int lane = threadIdx.x & 63;
    if (lane > 0 && lane < s.n) {
      const int64_t row = s.r0 + lane, up = max(ld_i(a.parent, row, a.parent_dtype), (int64_t)0);
      const int64_t t = ld_i(a.tokens, row, a.tokens_dtype);
      if (up < lane && t >= 0 && t < a.vocab) {
        parent = (int)up;
        token = (int)t;
        u = a.uniform[row];
        p = weight<T>(a.probs, (s.r0 + up) * a.probs_row_stride + t, a.probs_dtype);
        if (DRAFT) q = weight<T>(a.draft_probs, (s.r0 + up) * a.draft_row_stride + t, a.draft_dtype);
      }
    }
    r = p;
    kids = __ballot(parent == 0);
    w.path[0] = 0;
  }

  // On to the pass that comes next, with sum(pass) of the `have` ones made.
  template <class Sum>
  __device__ __forceinline__ void operator()(const dft_tree_accept_args& a, Walk& w, int have, Sum sum) {
    bool last = false;
    while (true) {
      if (waits) {
        if (pass == have) break;
        const double left = sum(pass++);
        w.f.by_sum[count - 1] = left > 0 ? 1 / left : 0;
        if (left > 0) r = rest / left;
        open = waits = false;
      }
      if (!kids || length >= a.path_cols) {
        last = true;
        break;
      }
      const int c = __ffsll((unsigned long long)kids) - 1;
      kids &= kids - 1;
      const int t = __builtin_amdgcn_readlane(token, c);
      bool stands;
      double take;  // what a refusal takes: of q, without a drafter's of r
      if constexpr (DRAFT) {
        const double now = gone || off >= 1 ? 0 : off > 0 ? q / (1 - off) : q;
        stands = of_lane(u, c) * of_lane(now, c) < of_lane(r, c);
        take = of_lane(gone ? 0 : q, c);
        rest = fmax(r - now, 0.0);
      } else {
        take = of_lane(gone ? 0 : p, c);
        stands = of_lane(u, c) * (1 - off) < take;
      }
      if (stands) {
        node = c;
        w.path[length++] = c;
        count = 0;
        off = 0;
        open = gone = false;
        r = p;
        kids = __ballot(parent == c);
        continue;
      }
      gone |= token == t;
      w.f.by_off[count] = off >= 1 ? 0 : 1 / (1 - off);
      w.f.token[count++] = t;
      off += take;
      if constexpr (DRAFT) {
        open = true;
        waits = kids;  // its sum decides about the next sibling
      }
    }
    w.f.count = count;
    w.node = node;
    w.length = length;
    w.pass = pass;
    w.open = open;
    w.last = last;
  }
};

// Four tokens of a row, from x on, of which those in [from, to) are there.
template <class T>
__device__ __forceinline__ f32x4 four(const void* p, int64_t at, int dt, int x, int from, int to, bool whole) {
  if constexpr (sizeof(T) > 1) {
    if (whole && x >= from && x + 4 <= to) {
      typedef T T4 __attribute__((ext_vector_type(4)));
      return __builtin_convertvector(*reinterpret_cast<const T4*>(static_cast<const T*>(p) + at + x), f32x4);
    }
  }
  f32x4 r = {};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (x + e < from || x + e >= to) continue;
    if constexpr (sizeof(T) > 1)
      r[e] = (float)static_cast<const T*>(p)[at + x + e];
    else
      r[e] = ld_f(p, at + x + e, dt);
  }
  return r;
}
// How far in front of a piece of four element `at` is; -1 where pieces are of no use.
template <class T>
__device__ __forceinline__ int in_piece(const void* p, int64_t at) {
  if constexpr (sizeof(T) == 1) return -1;
  return (int)((reinterpret_cast<uintptr_t>(static_cast<const T*>(p) + at) / sizeof(T)) & 3);
}

// This thread's part of a pass over tokens [from, to) of a row by `threads`
// threads: the tokens x(0) .. x(15) and what is left of each, handed to `take` in
// turn, sixteen at a time.  The reductions are products with 1 / (1 - off) and 1
// / sum, two roundings of 2^-53 beside the quotients of the walk.
template <bool DRAFT, class T, class Take>
__device__ __forceinline__ void pass_over(const dft_tree_accept_args& a, int64_t row, const Refused& f, int count, bool open, int from,
                                          int to, int thread, int threads, Take take) {
  const int64_t p_at = row * a.probs_row_stride, q_at = row * a.draft_row_stride;
  const bool drawn = DRAFT && count;
  int lead = in_piece<T>(a.probs, p_at + from);
  bool whole = lead >= 0;
  if (drawn) whole &= lead == in_piece<T>(a.draft_probs, q_at + from);
  lead = max(lead, 0);
  for (int x0 = from - lead + 4 * thread; x0 < to; x0 += 16 * threads) {
    f32x4 p[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = x0 + 4 * i * threads;
      p[i] = four<T>(a.probs, p_at, a.probs_dtype, x, from, to, whole);
      q[i] = drawn ? four<T>(a.draft_probs, q_at, a.draft_dtype, x, from, to, whole) : f32x4{};
    }
    double r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      r[i] = p[i / 4][i % 4] > 0 ? (double)p[i / 4][i % 4] : 0.0;
      if (DRAFT) q[i / 4][i % 4] = q[i / 4][i % 4] > 0 ? q[i / 4][i % 4] : 0.f;
    }
    for (int j = 0; j < count; ++j) {
      const double by_sum = !DRAFT || (j == count - 1 && open) ? 1 : f.by_sum[j];
      if (DRAFT && by_sum > 0) {
        const double by_off = f.by_off[j];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = fmax(r[i] - (double)q[i / 4][i % 4] * by_off, 0.0) * by_sum;
      }
      const int at = f.token[j] - x0;  // the refused one: out of q, or without a drafter's out of r
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool is = at == 4 * (i / 4) * threads + i % 4;
        if constexpr (DRAFT)
          q[i / 4][i % 4] = is ? 0.f : q[i / 4][i % 4];
        else
          r[i] = is ? 0 : r[i];
      }
    }
    take(r, [&](int i) { return x0 + 4 * (i / 4) * threads + i % 4; });
  }
}
// r's sum and its last token of any weight
template <bool DRAFT, class T>
__device__ __forceinline__ void add_up(const dft_tree_accept_args& a, int64_t row, const Refused& f, int count, bool open, int from,
                                       int to, int thread, int threads, double& sum, int& top) {
  sum = 0;
  top = -1;
  pass_over<DRAFT, T>(a, row, f, count, open, from, to, thread, threads, [&](const double(&r)[16], auto x) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sum += r[i];
      if (r[i] > 0) top = x(i);
    }
  });
}

// One pass of every request's, in slices.
template <bool DRAFT, class T>
__global__ void __launch_bounds__(kPass) pass_kernel(const dft_tree_accept_args a, Work work, int round) {
  __shared__ Walk w;
  __shared__ double sums[kPass / 64];
  __shared__ int tops[kPass / 64];
  const int b = blockIdx.x / work.slices, slice = blockIdx.x - b * work.slices, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const packed::Span s = packed::span_of(a.cu_seqlens, a.rows, a.n_nodes, b);
  if (s.n <= 0) return;
  // (each round's words are read by the next one: this one's slices start at any time)
  if (round && work.done[(round - 1) * a.batch + b]) {
    if (slice == 0 && tid == 0) work.done[round * a.batch + b] = 1;
    return;
  }
  auto sum_of = [&](int pass) {
    return wave_sum(lane < work.slices ? work.sums[((int64_t)pass * a.batch + b) * kSlices + lane] : 0.0);
  };
  if (wave == 0) Walker<DRAFT, T>(a, s, w)(a, w, round, sum_of);
  __syncthreads();
  const int from = min(slice * work.length, a.vocab), to = min(from + work.length, a.vocab);
  double sum;
  int top;
  add_up<DRAFT, T>(a, s.r0 + w.node, w.f, w.f.count, w.open, from, to, tid, kPass, sum, top);
  sum = wave_sum(sum);
  top = wave_max(top);
  if (lane == 0) sums[wave] = sum, tops[wave] = top;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kPass / 64; ++i) sum += sums[i], top = max(top, tops[i]);
    const int64_t at = ((int64_t)round * a.batch + b) * kSlices + slice;
    work.sums[at] = sum;
    work.tops[at] = top;
  }
  if (slice == 0) {
    if (tid == 0) work.done[round * a.batch + b] = w.last;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(&w);
    uint32_t* to = reinterpret_cast<uint32_t*>(work.walks + b);
    for (int i = tid; i < (int)(sizeof(Walk) / 4); i += kPass) to[i] = from[i];
  }
}

// The sum of the threads' values up to this one's, in thread order.
__device__ __forceinline__ double scan(double x, double* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(x, o);
    if (lane >= o) x += up;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  double ahead = 0;
  for (int i = 0; i < wave; ++i) ahead += waves[i];
  return ahead + x;
}

// The next token and the path, a workgroup a request.
template <bool DRAFT, class T>
__global__ void __launch_bounds__(kLast) last_kernel(const dft_tree_accept_args a, Work work, int rounds) {
  __shared__ Walk w;
  __shared__ double sums[kSlices], extra[kNodes], waves[kWaves], upto_all;
  __shared__ int tops[kSlices];
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // fetched side by side, whether there is a use for it or not: the walk, every round's sums, the random number
  constexpr int kWords = sizeof(Walk) / 4;
  static_assert(kWords <= kLast && kRounds * kSlices <= kLast);
  const double last = a.last[b];
  double slice_sum = 0;
  int slice_top = -1, done = 0;
  uint32_t word = 0;
  if (rounds) {
    done = work.done[(rounds - 1) * a.batch + b];
    if (tid < kWords) word = reinterpret_cast<const uint32_t*>(work.walks + b)[tid];
    if (tid < rounds * kSlices && lane < work.slices) {
      const int64_t at = ((int64_t)wave * a.batch + b) * kSlices + lane;
      slice_sum = work.sums[at];
      slice_top = work.tops[at];
    }
  }
  const packed::Span s = packed::span_of(a.cu_seqlens, a.rows, a.n_nodes, b);
  int* path = a.path + (int64_t)b * a.path_cols;
  int64_t* path_rows = a.path_rows + (int64_t)b * a.path_cols;
  int64_t token = -1;
  int length = 0;
  if (s.n > 0) {
    const int V = a.vocab;
    auto part_of = [&](int from, int to, int i) { return from + (int)((int64_t)(to - from) * i / kWaves); };
    // the sums of [from, to)'s equal parts, a wave each
    auto sum_up = [&](int from, int to, int count, bool open) {
      double sum;
      int top;
      add_up<DRAFT, T>(a, s.r0 + w.node, w.f, count, open, part_of(from, to, wave), part_of(from, to, wave + 1), lane, 64, sum, top);
      sum = wave_sum(sum);
      top = wave_max(top);
      __syncthreads();
      if (lane == 0) sums[wave] = sum, tops[wave] = top;
      __syncthreads();
    };
    auto total_of = [&](int parts) { return wave_sum(lane < parts ? sums[lane] : 0.0); };
    if (done) {
      if (tid < kWords) reinterpret_cast<uint32_t*>(&w)[tid] = word;
      __syncthreads();
    } else {
      auto sum_of = [&](int pass) {
        if (pass >= rounds) return extra[pass];
        return wave_sum(lane < work.slices ? work.sums[((int64_t)pass * a.batch + b) * kSlices + lane] : 0.0);
      };
      // passes that no round was left for are made here
      Walker<DRAFT, T> walker(a, s, w);
      for (int have = rounds;; ++have) {
        __syncthreads();
        if (wave == 0) walker(a, w, have, sum_of);
        __syncthreads();
        if (w.last) break;
        sum_up(0, V, w.f.count, w.open);
        const double sum = total_of(kWaves);
        if (tid == 0) extra[have] = sum;
      }
    }
    length = w.length;
    // the parts that the running sum is cut into, and whose sums are at hand
    int count = w.f.count, parts = kWaves;
    bool open = w.open, sliced = w.pass < rounds;
    if (sliced) {
      parts = work.slices;
      if (wave == w.pass) sums[lane] = slice_sum, tops[lane] = slice_top;
      __syncthreads();
    } else {
      sum_up(0, V, count, open);
    }
    double total = total_of(parts);
    // what reduces r to nothing is not taken from it
    while (!(total > 0) && count) {
      count = DRAFT ? count - 1 : 0;
      open = sliced = false;
      parts = kWaves;
      sum_up(0, V, count, open);
      total = total_of(parts);
    }
    if (total > 0) {
      const double target = last * total;
      double before = 0;
      int from = 0, to = V;
      while (token < 0) {
        // the part where the running sum passes the target, else the last of any weight (one of none has a sum that is
        // added up in another order, which may pass it first)
        double up = lane < parts ? sums[lane] : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double x = __shfl_up(up, o);
          if (lane >= o) up += x;
        }
        const uint64_t past = __ballot(lane < parts && sums[lane] > 0 && before + up > target);
        if (!past) {
          token = wave_max(lane < parts ? tops[lane] : -1);
          break;
        }
        const int part = __ffsll((unsigned long long)past) - 1;
        const double ahead = part ? __shfl(up, part - 1) : 0;
        const int first = sliced ? min(part * work.length, V) : part_of(from, to, part);
        to = sliced ? min(first + work.length, V) : part_of(from, to, part + 1);
        from = first;
        before += ahead;
        sliced = false;
        parts = kWaves;
        const int lead = max(in_piece<T>(a.probs, (s.r0 + w.node) * a.probs_row_stride + from), 0);
        if (lead + to - from > 16 * kLast) {
          sum_up(from, to, count, open);
          continue;
        }
        // few enough for one step: a piece of 4 tokens a thread, four times over, in order
        double part_sum[4] = {}, r4[16] = {};
        int x4 = 0;
        pass_over<DRAFT, T>(a, s.r0 + w.node, w.f, count, open, from, to, tid, kLast, [&](const double(&r)[16], auto x) {
          x4 = x(0);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            r4[i] = r[i];
            part_sum[i / 4] += r[i];
          }
        });
        if (tid == 0) found = V;
        int last_top = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const double upto = scan(part_sum[k], waves);
          // the first piece of any weight whose sum passes the target, and in it the token that does
          const uint64_t past = __ballot(before + upto > target && part_sum[k] > 0);
          if (past && lane == __ffsll((unsigned long long)past) - 1) {
            double c = before + (upto - part_sum[k]);
            int at = V;
            bool over = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool some = r4[4 * k + e] > 0;
              if (!over && some) at = x4 + 4 * k * kLast + e;
              c += r4[4 * k + e];
              over |= some && c > target;
            }
            atomicMin(&found, at);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r4[4 * k + e] > 0) last_top = x4 + 4 * k * kLast + e;
          if (tid == kLast - 1) upto_all = upto;
          __syncthreads();
          before += upto_all;
          if (found < V) break;
        }
        __syncthreads();
        token = found;
        if (token == V) {  // rounding: the last of any weight here
          last_top = wave_max(last_top);
          if (lane == 0) tops[wave] = last_top;
          __syncthreads();
          token = wave_max(lane < kWaves ? tops[lane] : -1);
        }
        break;
      }
    }
  }
  for (int c = tid; c < a.path_cols; c += kLast) {
    const int node = c < length ? w.path[c] : -1;
    path[c] = node;
    path_rows[c] = node < 0 ? -1 : s.r0 + node;
  }
  if (tid == 0) {
    a.path_len[b] = length;
    a.token[b] = token;
    if (a.status) a.status[b] = s.status | (s.n > 0 && token < 0 ? DFT_STATUS_WEIGHT : 0);
  }
}

// A pass for every refused child with a sibling behind it, and the last one: no
// more than there are children.  None over short rows, which a request's workgroup
// passes over as fast.  Trees of 16 nodes, us in a captured graph, without rounds
// and with: one request over 2000 tokens 10 and 11, drawn 9 and 15, 16000 11.5 and
// 11, 10 and 16, 64000 19 and 11, 55 and 29; 64 requests 11 and 12, 22 and 30,
// then 12 and 13, 26 and 34, then 24 and 18, 65 and 50; 500 requests 14 and 15, 35
// and 54, then 18 and 23, 49 and 74, then 37 and 45, 124 and 145.
int rounds_of(const dft_tree_accept_args& a) {
  if (a.vocab <= kShort) return 0;
  return a.draft_probs ? std::min(kRounds, std::max(a.n_nodes - 1, 1)) : 1;
}
// Slices such that a pass has some two thousand workgroups, of no less than 1024
// tokens.  (With one thousand the same 48 drawn trees took 56 us instead of 49, 64
// chains 30 instead of 32.)
Work work_of(const dft_tree_accept_args& a) {
  Work w = {};
  const int most = std::min(kSlices, std::max(1, 2048 / a.batch));
  w.length = std::max(1024, ((a.vocab + most - 1) / most + 1023) / 1024 * 1024);
  w.slices = std::max(1, (a.vocab + w.length - 1) / w.length);
  return w;
}

template <bool DRAFT, class T>
int launch(const dft_tree_accept_args& a, const Work& work, hipStream_t stream) {
  for (int round = 0; round < rounds_of(a); ++round)
    pass_kernel<DRAFT, T><<<(unsigned)(a.batch * work.slices), kPass, 0, stream>>>(a, work, round);
  last_kernel<DRAFT, T><<<a.batch, kLast, 0, stream>>>(a, work, rounds_of(a));
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}
template <class T>
int launch_type(const dft_tree_accept_args& a, const Work& work, hipStream_t stream) {
  return a.draft_probs ? launch<true, T>(a, work, stream) : launch<false, T>(a, work, stream);
}

}  // namespace

// (for either form: whether there is a drafter's distribution need not be known yet)
int64_t tree_accept_workspace(const dft_tree_accept_args* a) {
  return (int64_t)a->batch * (sizeof(Walk) + kRounds * (kSlices * (sizeof(double) + sizeof(int)) + sizeof(int)));
}

int launch_tree_accept(const dft_tree_accept_args* a, hipStream_t stream) {
  static_assert(sizeof(Walk) % 8 == 0);
  Work work = work_of(*a);
  const int64_t passes = (int64_t)kRounds * a->batch;
  work.walks = static_cast<Walk*>(a->workspace);
  work.sums = reinterpret_cast<double*>(work.walks + a->batch);
  work.tops = reinterpret_cast<int*>(work.sums + passes * kSlices);
  work.done = work.tops + passes * kSlices;
  if (a->draft_probs && a->draft_dtype != a->probs_dtype) return launch<true, uint8_t>(*a, work, stream);
  switch (a->probs_dtype) {
    case DFT_BF16: return launch_type<__bf16>(*a, work, stream);
    case DFT_F16: return launch_type<_Float16>(*a, work, stream);
    default: return launch_type<float>(*a, work, stream);
  }
}

}  // namespace dft
