// dft_tree_accept: which drafted tokens stand, and the token behind them.
//
// The nodes of a request are looked at once each, in index order: node i is
// examined where its parent is the node that the path stands at by then (a
// child's index is larger than its parent's, and siblings are taken in index
// order).  Sums are held in 64 bits: a sum of 10^5 probabilities in 32 bits
// moves one drawn token in some hundred over a border.
#include "packed.h"

namespace dft {
namespace {

constexpr int kNodes = 64, kWaves = 16, kThreads = 64 * kWaves;

__device__ __forceinline__ double weight(const void* p, int64_t at, int dt) {
  const float x = ld_f(p, at, dt);
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

// r at token x behind `count` refused ones; the last reduction's sum may not
// be known yet (`open`): it is not divided by.
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
      const double q = gone || f.off[j] >= 1 ? 0 : q0 / (1 - f.off[j]);
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

template <bool DRAFT>
__global__ void __launch_bounds__(kThreads) accept_kernel(const dft_tree_accept_args a) {
  __shared__ Refused f;
  __shared__ double sums[kWaves];
  __shared__ int some[kWaves];
  __shared__ double cum[kThreads];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const packed::Span s = packed::span_of(a.cu_seqlens, a.rows, a.n_nodes, b);
  int64_t row = s.r0;  // of the node that the path stands at
  const int V = a.vocab;

  auto at = [&](int x, int count, bool open) {
    const double p = weight(a.probs, row * a.probs_row_stride + x, a.probs_dtype);
    const double q = DRAFT && count ? weight(a.draft_probs, row * a.draft_row_stride + x, a.draft_dtype) : 0;
    return left_at<DRAFT>(p, q, x, f, count, open);
  };
  // the sum of r over [from, to), in all threads; the waves take a sixteenth each
  auto slice = [&](int from, int to, int w) { return from + (int)((int64_t)(to - from) * w / kWaves); };
  auto sum_up = [&](int from, int to, int count, bool open) {
    double sum = 0;
    int top = -1;
    for (int x = slice(from, to, wave) + lane; x < slice(from, to, wave + 1); x += 64) {
      const double r = at(x, count, open);
      sum += r;
      if (r > 0) top = x;
    }
    sum = wave_sum(sum);
    for (int o = 32; o; o >>= 1) top = max(top, __shfl_xor(top, o));
    __syncthreads();
    if (lane == 0) sums[wave] = sum, some[wave] = top;
    __syncthreads();
    double total = 0;
    for (int w = 0; w < kWaves; ++w) total += sums[w];
    return total;
  };

  int node = 0, length = s.n > 0 ? 1 : 0;
  int* path = a.path + (int64_t)b * a.path_cols;
  int64_t* path_rows = a.path_rows + (int64_t)b * a.path_cols;
  for (int c = tid; c < a.path_cols; c += kThreads) {
    path[c] = c == 0 && length ? 0 : -1;
    path_rows[c] = c == 0 && length ? row : -1;
  }
  __syncthreads();
  if (tid == 0) f.count = 0, f.off[0] = 0;
  __syncthreads();
  for (int i = 1; i < s.n && length < a.path_cols; ++i) {
    const int64_t ri = s.r0 + i;
    if (max(ld_i(a.parent, ri, a.parent_dtype), (int64_t)0) != node) continue;
    const int64_t t = ld_i(a.tokens, ri, a.tokens_dtype);
    if (t < 0 || t >= V) continue;
    const double u = a.uniform[ri];
    const int count = f.count;
    const double off = f.off[count];
    bool gone = false;
    for (int j = 0; j < count; ++j) gone |= f.token[j] == t;
    const double r = at((int)t, count, false);
    bool stands;
    double take;  // what a refusal takes: of q, without a drafter's of r
    if constexpr (DRAFT) {
      const double q0 = weight(a.draft_probs, row * a.draft_row_stride + t, a.draft_dtype);
      stands = u * (gone || off >= 1 ? 0 : q0 / (1 - off)) < r;
      take = gone ? 0 : q0;
    } else {
      stands = u * (1 - off) < r;
      take = r;
    }
    __syncthreads();
    if (stands) {
      node = i;
      row = ri;
      if (tid == 0) {
        path[length] = i;
        path_rows[length] = ri;
        f.count = 0, f.off[0] = 0;
      }
      ++length;
    } else {
      if (tid == 0) {
        f.token[count] = (int)t;
        f.off[count + 1] = off + take;
        f.count = count + 1;
      }
      if constexpr (DRAFT) {
        __syncthreads();
        const double sum = sum_up(0, V, count + 1, true);
        if (tid == 0) f.sum[count] = sum;
      }
    }
    __syncthreads();
  }

  int64_t token = -1;
  if (s.n > 0) {
    // the last refusal changes nothing where it leaves nothing
    int count = f.count;
    if (DRAFT) {
      while (count && !(f.sum[count - 1] > 0)) --count;
    }
    double total = sum_up(0, V, count, false);
    if (!DRAFT && count && !(total > 0)) total = sum_up(0, V, count = 0, false);
    double target = (double)a.last[b] * total, before = 0;
    int from = 0, to = V;
    if (total > 0) {
      while (true) {
        // the part where the running sum passes the target, or the last of any weight
        int part = -1, last = -1;
        double ahead = before, start = before;
        for (int w = 0; w < kWaves; ++w) {
          if (some[w] >= 0) last = w;
          if (part < 0 && ahead + sums[w] > target) part = w, start = ahead;
          ahead += sums[w];
        }
        if (part < 0) {
          token = some[last];
          break;
        }
        const int f1 = slice(from, to, part), t1 = slice(from, to, part + 1);
        from = f1, to = t1, before = start;
        if (to - from <= kThreads) {
          __syncthreads();
          cum[tid] = from + tid < to ? at(from + tid, count, false) : 0;
          __syncthreads();
          double c = before;
          for (int x = from; x < to; ++x) {
            const double r = cum[x - from];
            c += r;
            if (r > 0) token = x;
            if (c > target) break;
          }
          break;
        }
        sum_up(from, to, count, false);
      }
    }
  }
  if (tid == 0) {
    a.path_len[b] = length;
    a.token[b] = token;
    if (a.status) a.status[b] = s.status | (s.n > 0 && token < 0 ? DFT_STATUS_WEIGHT : 0);
  }
}

}  // namespace

int64_t tree_accept_workspace(const dft_tree_accept_args*) { return 0; }

int launch_tree_accept(const dft_tree_accept_args* a, hipStream_t stream) {
  if (a->draft_probs)
    accept_kernel<true><<<a->batch, kThreads, 0, stream>>>(*a);
  else
    accept_kernel<false><<<a->batch, kThreads, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace dft
