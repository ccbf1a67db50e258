// dft_tree_accept: which drafted tokens stand, and the token behind them.
//
// The walk from the root needs of every node only two values, p and q at its
// token in its parent's rows, which are fetched for all nodes at once; the walk
// itself is a wave's work on them.  What takes time is whole rows: the sum of
// max(r - q, 0) where a refused child has another sibling, and r's running sum
// at the end.  Such a pass over a row is cut into slices, a workgroup each.  A
// launch does one pass for every request, whatever it is of that request's; the
// next one walks again, with the sums there are, to the next pass.  Without the
// drafter's probabilities the first pass is the last; with them kRounds launches
// are made, and what is still open is done by the request's workgroup alone in
// the last launch, which finds the token.
//
// Sums are held in 64 bits: a sum of 10^5 probabilities in 32 bits moves one
// drawn token in some hundred over a border.  They are added up in one order.
#include <algorithm>

#include "packed.h"

namespace dft {
namespace {

constexpr int kNodes = 64, kSlices = 64, kRounds = 3;
constexpr int kPass = 256, kLast = 1024, kWaves = kLast / 64;  // threads of a pass and of the last launch

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
  double off[kNodes + 1];  // mass of the tokens in front of this one
  double sum[kNodes];      // of the weights left behind it (drafter's distribution given)
};

// r at token x behind `count` refused ones; `open`: the last one's sum is not
// known, and not divided by.
template <bool DRAFT>
__device__ __forceinline__ double left_at(double p, double q0, int x, const Refused& f, int count, bool open) {
  if constexpr (!DRAFT) {
    for (int j = 0; j < count; ++j)
      if (f.token[j] == x) return 0;
    return p;
  } else {
    double r = p;
    bool gone = false;
    for (int j = 0; j < count; ++j) {
      const double off = f.off[j];
      const double q = gone || off >= 1 ? 0 : off > 0 ? q0 / (1 - off) : q0;
      const double rest = fmax(r - q, 0.0);
      if (j == count - 1 && open)
        r = rest;
      else if (f.sum[j] > 0)
        r = rest / f.sum[j];
      gone |= f.token[j] == x;
    }
    return r;
  }
}

__device__ __forceinline__ double wave_sum(double x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ int wave_max(int x) {
  for (int o = 32; o; o >>= 1) x = max(x, __shfl_xor(x, o));
  return x;
}

struct Work {
  double* sums;  // [round][batch][kSlices]
  int* tops;     // the same: the last token of any weight, -1 for none
  int slices, length;  // of a pass; tokens of a slice
};

// A request's walk as far as it goes, in the LDS.
struct Walk {
  Refused f;
  int path[kNodes];
  int node, length, pass;  // where the path stands, its nodes, the pass that comes next
  bool open, last;         // whether that is of the last refusal, and the walk's last
};

// By the first wave, a node a lane.  sum(pass): an earlier round's, `have` of them.
template <bool DRAFT, class T, class Sum>
__device__ __forceinline__ void walk(const dft_tree_accept_args& a, const packed::Span& s, Walk& w, int have, Sum sum) {
  const int lane = threadIdx.x & 63;
  int parent = -1, token = 0;
  double u = 0, p = 0, q = 0;
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
  // every lane keeps the same state, and writes the same to the LDS
  int node = 0, length = s.n > 0, count = 0, pass = 0;
  bool open = false, last = false;
  double off = 0;
  w.path[0] = 0;
  w.f.off[0] = 0;
  uint64_t kids = __ballot(parent == 0);
  while (true) {
    if (!kids || length >= a.path_cols) {
      last = true;
      break;
    }
    const int c = __ffsll((unsigned long long)kids) - 1;
    kids &= kids - 1;
    const int t = __shfl(token, c);
    const double uc = __shfl(u, c), pc = __shfl(p, c), qc = __shfl(q, c);
    bool gone = false;
    for (int j = 0; j < count; ++j) gone |= w.f.token[j] == t;
    const double r = left_at<DRAFT>(pc, qc, t, w.f, count, false);
    bool stands;
    double take;  // what a refusal takes: of q, without a drafter's of r
    if constexpr (DRAFT) {
      stands = uc * (gone || off >= 1 ? 0 : off > 0 ? qc / (1 - off) : qc) < r;
      take = gone ? 0 : qc;
    } else {
      stands = uc * (1 - off) < r;
      take = r;
    }
    if (stands) {
      node = c;
      w.path[length++] = c;
      count = 0;
      off = 0;
      open = false;
      kids = __ballot(parent == c);
      continue;
    }
    w.f.token[count++] = t;
    off += take;
    w.f.off[count] = off;
    if constexpr (DRAFT) {
      open = true;
      if (kids) {  // its sum decides about the next sibling
        if (pass == have) break;
        w.f.sum[count - 1] = sum(pass++);
        open = false;
      }
    }
  }
  w.f.count = count;
  w.node = node;
  w.length = length;
  w.pass = pass;
  w.open = open;
  w.last = last;
}

// r's sum over [from, to) and its last token of any weight, by `threads` threads:
// this thread's part.
template <bool DRAFT, class T>
__device__ __forceinline__ void add_up(const dft_tree_accept_args& a, int64_t row, const Refused& f, int count, bool open, int from,
                                       int to, int thread, int threads, double& sum, int& top) {
  constexpr int kAhead = 8;
  sum = 0;
  top = -1;
  const int64_t p_at = row * a.probs_row_stride, q_at = row * a.draft_row_stride;
  for (int x = from + thread; x < to; x += kAhead * threads) {
    double p[kAhead], q[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = min(x + i * threads, to - 1);
      p[i] = weight<T>(a.probs, p_at + at, a.probs_dtype);
      q[i] = DRAFT && count ? weight<T>(a.draft_probs, q_at + at, a.draft_dtype) : 0;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = x + i * threads;
      const double r = at < to ? left_at<DRAFT>(p[i], q[i], at, f, count, open) : 0;
      sum += r;
      if (r > 0) top = at;
    }
  }
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
  auto sum_of = [&](int pass) {
    return wave_sum(lane < work.slices ? work.sums[((int64_t)pass * a.batch + b) * kSlices + lane] : 0.0);
  };
  if (wave == 0) walk<DRAFT, T>(a, s, w, round, sum_of);
  __syncthreads();
  if (w.pass != round) return;  // its last pass has been made
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
}

// The next token and the path, a workgroup a request.
template <bool DRAFT, class T>
__global__ void __launch_bounds__(kLast) last_kernel(const dft_tree_accept_args a, Work work, int rounds) {
  __shared__ Walk w;
  __shared__ double sums[kSlices], extra[kRounds > kNodes ? kRounds : kNodes];
  __shared__ int tops[kSlices];
  __shared__ double r_of[kLast];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const packed::Span s = packed::span_of(a.cu_seqlens, a.rows, a.n_nodes, b);
  int* path = a.path + (int64_t)b * a.path_cols;
  int64_t* path_rows = a.path_rows + (int64_t)b * a.path_cols;
  int64_t token = -1;
  int length = 0;
  if (s.n > 0) {
    const int V = a.vocab;
    auto part_of = [&](int from, int to, int i) { return from + (int)((int64_t)(to - from) * i / kWaves); };
    // the sums of [from, to)'s sixteenths, a wave each
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
    auto total_of = [&](int parts) {
      double total = 0;
      for (int i = 0; i < parts; ++i) total += sums[i];
      return total;
    };
    auto sum_of = [&](int pass) {
      if (pass >= rounds) return extra[pass];
      return wave_sum(lane < work.slices ? work.sums[((int64_t)pass * a.batch + b) * kSlices + lane] : 0.0);
    };
    // passes that no round was left for are made here
    for (int have = rounds;; ++have) {
      __syncthreads();
      if (wave == 0) walk<DRAFT, T>(a, s, w, have, sum_of);
      __syncthreads();
      if (w.last) break;
      sum_up(0, V, w.f.count, w.open);
      const double sum = total_of(kWaves);
      __syncthreads();
      if (tid == 0) extra[have] = sum;
    }
    length = w.length;
    // the parts that the running sum is cut into, and whose sums are at hand
    int count = w.f.count, parts = kWaves;
    bool open = w.open, sliced = w.pass < rounds;
    if (sliced) {
      parts = work.slices;
      if (tid < parts) {
        const int64_t at = ((int64_t)w.pass * a.batch + b) * kSlices + tid;
        sums[tid] = work.sums[at];
        tops[tid] = work.tops[at];
      }
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
      const double target = (double)a.last[b] * total;
      double before = 0;
      int from = 0, to = V;
      while (true) {
        // the part where the running sum passes the target, else the last of any weight
        int part = -1, last = 0;
        double ahead = before, start = before;
        for (int i = 0; i < parts; ++i) {
          if (tops[i] >= 0) last = i;
          if (part < 0 && ahead + sums[i] > target) part = i, start = ahead;
          ahead += sums[i];
        }
        if (part < 0) {
          token = tops[last];
          break;
        }
        const int first = sliced ? min(part * work.length, V) : part_of(from, to, part);
        to = sliced ? min(first + work.length, V) : part_of(from, to, part + 1);
        from = first;
        before = start;
        sliced = false;
        parts = kWaves;
        if (to - from <= 64) break;
        sum_up(from, to, count, open);
      }
      if (token < 0) {  // 64 of them at most: by one wave
        double r = 0;
        if (lane < to - from) {
          int top;
          add_up<DRAFT, T>(a, s.r0 + w.node, w.f, count, open, from + lane, from + lane + 1, 0, 1, r, top);
        }
        double c = before;
        for (int x = 0; x < to - from; ++x) {  // in order
          const double rx = __shfl(r, x);
          c += rx;
          if (rx > 0) token = from + x;
          if (c > target) break;
        }
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

int rounds_of(const dft_tree_accept_args& a) { return a.draft_probs ? kRounds : 1; }
// Slices such that a pass has some thousand workgroups, of no less than 1024 tokens.
Work work_of(const dft_tree_accept_args& a) {
  Work w = {};
  const int most = std::min(kSlices, std::max(1, 1024 / a.batch));
  w.length = std::max(1024, (a.vocab + most - 1) / most);
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
  return (int64_t)kRounds * a->batch * kSlices * (int64_t)(sizeof(double) + sizeof(int));
}

int launch_tree_accept(const dft_tree_accept_args* a, hipStream_t stream) {
  Work work = work_of(*a);
  work.sums = static_cast<double*>(a->workspace);
  work.tops = reinterpret_cast<int*>(work.sums + (int64_t)kRounds * a->batch * kSlices);
  if (a->draft_probs && a->draft_dtype != a->probs_dtype) return launch_type<uint8_t>(*a, work, stream);
  switch (a->probs_dtype) {
    case DFT_BF16: return launch_type<__bf16>(*a, work, stream);
    case DFT_F16: return launch_type<_Float16>(*a, work, stream);
    default: return launch_type<float>(*a, work, stream);
  }
}

}  // namespace dft
