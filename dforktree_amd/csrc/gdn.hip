// dft_prompt_gdn: the gated delta rule over packed prompts and single tokens.
//
// Per v head and row, q and k normalised, q scaled:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q
// Single tokens: row by row, gdn_rows_kernel.  Prompts: in chunks of 64 rows,
// for whose rows i and j, G the running sum of g within the chunk, K and Q the
// raw rows, rk and rq what normalises (and scales) them:
//   A_ij = beta_i rk_i rk_j (k_i . k_j) e^(G_i - G_j)  (j < i),  X = (I + A)^-1
//   P_ij = rq_i rk_j (q_i . k_j) e^(G_i - G_j)         (j <= i)
//   W = beta (V - e^G rk (K S)),  U = X W
//   O = e^G rq (Q S) + P U
//   S <- e^G_63 S + K^T (e^(G_63 - G) rk U)
// gdn_chunk_kernel forms what needs no state, X and P, for all chunks at once,
// gdn_scan_kernel takes the states through the chunks.  The raw rows are bf16,
// so that K, Q and K^T are exact operands of bf16 products; what is not (S, X,
// P, W, U) goes in as a pair hi + lo, 2^-16 relative at most, a product of two
// pairs without lo * lo.  (States are handed on in fp32 from chunk to chunk
// and are held to it: one bf16 factor would leave 2^-9 in them.)
#include <algorithm>

#include "packed.h"

namespace dft {
namespace {

using namespace packed;

constexpr int kD = 128;

// g and beta of one row and head
struct Gate {
  float g, beta;
};
__device__ __forceinline__ Gate gate_of(const dft_prompt_gdn_args& a, int64_t row, int h) {
  const float rate = a.neg_exp_A ? a.neg_exp_A[h] : -expf(ld_f(a.A_log, h, a.A_log_dtype));
  const float x = ld_f(a.a, row * a.a_row_stride + h, a.a_dtype) + ld_f(a.dt_bias, h, a.dt_bias_dtype);
  const float soft = x > 20.f ? x : log1pf(expf(x));
  return {rate * soft, 1.f / (1.f + expf(-ld_f(a.b, row * a.b_row_stride + h, a.b_dtype)))};
}

// The sum over a row of 16 lanes, in all of them.
__device__ __forceinline__ float sum16(float x) {
  x += __shfl_xor(x, 1);
  x += __shfl_xor(x, 2);
  x += __shfl_xor(x, 4);
  x += __shfl_xor(x, 8);
  return x;
}

// ---- row by row ------------------------------------------------------------
// A workgroup of four waves keeps V value columns of one head's state in
// registers: 16 lanes a column, 8 keys a lane (4 i .. and 64 + 4 i ..), so that
// a wave's access covers whole columns and both sums over the keys stay within
// 16 lanes.
template <int V, bool VEC>
__global__ void __launch_bounds__(256) gdn_rows_kernel(const dft_prompt_gdn_args a) {
  constexpr int kSplit = kD / V, kPass = V / 16;
  const int64_t x = blockIdx.x;
  if (x == 0 && a.status)
    for (int b = threadIdx.x; b < a.batch; b += 256)
      a.status[b] = span_of(a, b).status | slot_of(a.state_indices, a.state_indices_dtype, a.initial, a.slots, b).status;
  const int per = a.hv * kSplit;
  const int b = (int)(x / per), r = (int)(x - (int64_t)b * per), h = r / kSplit, part = r - h * kSplit;
  const Span s = span_of(a, b);
  if (s.n <= 0) return;
  const Slot slot = slot_of(a.state_indices, a.state_indices_dtype, a.initial, a.slots, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, quad = lane >> 4;
  const int kh = h / (a.hv / a.hk), v0 = part * V + wave * (V / 4) + quad;  // + 4 pass: the lane's value columns

  float S[kPass][8];
  float* state = a.state + slot.at * a.state_slot_stride + h * a.state_h_stride;
  auto at = [&](int p, int e) { return (4 * i + (e & 3) + (e >> 2) * 64) * a.state_k_stride + (v0 + 4 * p) * a.state_v_stride; };
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    if (!slot.initial) {
#pragma unroll
      for (int e = 0; e < 8; ++e) S[p][e] = 0;
    } else if constexpr (VEC) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(state + at(p, 4 * y));
#pragma unroll
        for (int e = 0; e < 4; ++e) S[p][4 * y + e] = w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) S[p][e] = state[at(p, e)];
    }
  }
  const uint16_t* y = static_cast<const uint16_t*>(a.y);
  for (int t = 0; t < s.n; ++t) {
    const int64_t row = s.r0 + t;
    const uint16_t* yr = y + row * a.y_row_stride;
    float q[8], k[8], qq = 0, kk = 0, qk = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = kh * kD + 4 * i + (e & 3) + (e >> 2) * 64;
      q[e] = bf16_bits_to_f32(yr[c]);
      k[e] = bf16_bits_to_f32(yr[a.hk * kD + c]);
      qq = fmaf(q[e], q[e], qq);
      kk = fmaf(k[e], k[e], kk);
    }
    const float rq = a.scale / sqrtf(sum16(qq) + 1e-6f), rk = 1.f / sqrtf(sum16(kk) + 1e-6f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] *= rq;
      k[e] *= rk;
      qk = fmaf(q[e], k[e], qk);
    }
    qk = sum16(qk);
    const Gate g = gate_of(a, row, h);
    const float decay = expf(g.g);
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      float kS = 0, qS = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        S[p][e] *= decay;
        kS = fmaf(k[e], S[p][e], kS);
        qS = fmaf(q[e], S[p][e], qS);
      }
      kS = sum16(kS);
      qS = sum16(qS);
      const int v = v0 + 4 * p;
      const float u = g.beta * (bf16_bits_to_f32(yr[2 * a.hk * kD + h * kD + v]) - kS);
#pragma unroll
      for (int e = 0; e < 8; ++e) S[p][e] = fmaf(k[e], u, S[p][e]);
      if (i == p) store(a.o, row * a.o_row_stride + h * a.o_h_stride + v, a.o_dtype, fmaf(qk, u, qS));
    }
  }
  if (slot.at < 0) return;
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    if constexpr (VEC) {
#pragma unroll
      for (int y = 0; y < 2; ++y)
        *reinterpret_cast<f32x4*>(state + at(p, 4 * y)) = f32x4{S[p][4 * y], S[p][4 * y + 1], S[p][4 * y + 2], S[p][4 * y + 3]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) state[at(p, e)] = S[p][e];
    }
  }
}

// ---- chunks of 64 rows -----------------------------------------------------
// Fragments of v_mfma_f32_16x16x32_bf16: lane l holds 8 elements of row (of the
// left operand; column of the right one) l % 16, the terms 8 (l / 16) .. of a
// step of 32; of the result column l % 16, rows 4 (l / 16) ...  A product may
// take its terms in any order, so what a result leaves in a lane is the next
// product's operand without an exchange wherever both operands agree on it:
// terms that are chunk rows stand in the order
//   32 s + 16 h + 4 g + e  at place  32 s + 8 g + 4 h + e.
constexpr int kChunk = 64, kXcds = 8;
constexpr int kFragment = 1024;  // bytes: 64 lanes x 16
// Of X - I and P, whose upper halves are zero, the row tile m (of 16) has steps
// 0 .. m / 2: six fragments, X's in three parts, P's in two behind them.  P's row
// tiles 0 and 1 have a fragment of zeros for their other step, so that all
// waves do the same (loads whose use depends on the wave are waited for too early).
constexpr int kTriangle = 6 * 5 * kFragment;
constexpr int kCoef = 5 * kChunk * 4;  // of the rows: beta, e^G rk beta, e^(G_63 - G) rk, e^G_63 (of all), e^G rq
constexpr int kHead = kTriangle + kCoef + kFragment, kKeys = 16 * kFragment;
__device__ __forceinline__ int x_at(int m, int s) { return (m < 2 ? m : 2 * m - 2 + s) * 3 * kFragment; }
__device__ __forceinline__ int p_at(int m, int s) { return 18 * kFragment + (m < 2 ? m : 2 * m - 2 + s) * 2 * kFragment; }

// Row i of K^T's row tile m: such that the lane that holds rows 4 g .. of the
// results of tiles 2 w and 2 w + 1 has the keys 32 w + 8 g .., which are its
// terms of step w.
__device__ __forceinline__ int key_of(int m, int i) { return 32 * (m / 2) + 8 * (i / 4) + 4 * (m % 2) + i % 4; }

struct Work {
  char* heads;  // [tile][hv][kHead]: X, P, the rows' factors
  char* keys;   // [tile][hk][kKeys]: K^T
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// x = p[0] + p[1] + ..., each the bf16 nearest to what is left
template <int N>
struct Parts4 {
  uint64_t p[N];
};
template <int N>
__device__ __forceinline__ Parts4<N> split4(f32x4 x) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  Parts4<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bf16x4 h = __builtin_convertvector(x, bf16x4);
    r.p[i] = __builtin_bit_cast(uint64_t, h);
    if (i + 1 < N) x -= __builtin_convertvector(h, f32x4);
  }
  return r;
}
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

// The part of a chunk and v head that needs no state: a workgroup of four
// waves, wave w for rows 16 w ...  X row block by row block from X (I + A) = I:
// diagonal blocks by substitution (their powers would lose what equal keys
// leave of 32 bits), then X_ij = -(sum_(j<m<=i) X_im A_mj) X_jj in fp32
// products, transposed, so that each result is the next one's operand and the
// last the fragment that is stored.
__global__ void __launch_bounds__(256) gdn_chunk_kernel(const dft_prompt_gdn_args a, Work work) {
  constexpr int kKRow = kD + 8, kARow = kChunk + 4;
  __shared__ __attribute__((aligned(16))) uint16_t keys[kChunk][kKRow];
  __shared__ __attribute__((aligned(16))) float A[kChunk][kARow];
  __shared__ __attribute__((aligned(16))) float G[kChunk], beta[kChunk], rks[kChunk], rqs[kChunk];
  const int64_t tile = blockIdx.x / a.hv;
  const int h = (int)(blockIdx.x - tile * a.hv), group = a.hv / a.hk, kh = h / group;
  const int b = find_tile<256>(a, tile, kChunk);
  if (b < 0) return;
  const Span s = span_of(a, b);
  const int t0 = (int)(tile - first_tile(s.r0, b, kChunk)) * kChunk, n = min(s.n - t0, kChunk);
  const int64_t r0 = s.r0 + t0;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;

  // rows past the request's last: zeros
  bf16x8 q[4], k[4];
  float qq = 0, kk = 0;
  const int mine = 16 * w + l16;
  const uint16_t* row = static_cast<const uint16_t*>(a.y) + (r0 + min(mine, n - 1)) * a.y_row_stride + kh * kD + 8 * g;
  u32x4 qw[4], kw[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    qw[j] = *reinterpret_cast<const u32x4*>(row + 32 * j);
    kw[j] = *reinterpret_cast<const u32x4*>(row + a.hk * kD + 32 * j);
  }
  Gate gate = {};
  float sum = 0, all = 0;
  if (w == 0) {  // the gates, a row a lane, G in log2 units
    gate = gate_of(a, r0 + min(lane, n - 1), h);
    if (lane >= n) gate.g = gate.beta = 0;
    sum = gate.g * 1.4426950408889634f;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float up = __shfl_up(sum, o);
      if (lane >= o) sum += up;
    }
    all = __shfl(sum, 63);
    G[lane] = sum;
    beta[lane] = gate.beta;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (mine >= n) qw[j] = kw[j] = u32x4{};
    q[j] = __builtin_bit_cast(bf16x8, qw[j]);
    k[j] = __builtin_bit_cast(bf16x8, kw[j]);
    *reinterpret_cast<u32x4*>(&keys[mine][32 * j + 8 * g]) = kw[j];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qq = fmaf((float)q[j][e], (float)q[j][e], qq);
      kk = fmaf((float)k[j][e], (float)k[j][e], kk);
    }
  }
  qq += __shfl_xor(qq, 16);
  kk += __shfl_xor(kk, 16);
  qq += __shfl_xor(qq, 32);
  kk += __shfl_xor(kk, 32);
  const float rq = a.scale / sqrtf(qq + 1e-6f);
  if (g == 0) {
    rks[mine] = 1.f / sqrtf(kk + 1e-6f);
    rqs[mine] = rq;
  }
  __syncthreads();

  char* out = work.heads + (tile * a.hv + h) * kHead;
  if (w == 0) {
    float* coef = reinterpret_cast<float*>(out + kTriangle);
    const float e = __builtin_amdgcn_exp2f(sum), rk = rks[lane];
    coef[lane] = gate.beta;
    coef[kChunk + lane] = lane < n ? e * rk * gate.beta : 0;
    coef[2 * kChunk + lane] = lane < n ? __builtin_amdgcn_exp2f(all - sum) * rk : 0;
    coef[3 * kChunk + lane] = __builtin_amdgcn_exp2f(all);
    coef[4 * kChunk + lane] = e * rqs[lane];
    *reinterpret_cast<u32x4*>(out + kTriangle + kCoef + 16 * lane) = u32x4{};
  }

  // A into the LDS, P to its place: Gram tiles of the wave's rows with those of tiles j <= w, K K^T and (Q K^T)^T
  const f32x4 Gi = *reinterpret_cast<const f32x4*>(&G[16 * w + 4 * g]);
  const f32x4 bi = *reinterpret_cast<const f32x4*>(&beta[16 * w + 4 * g]) * *reinterpret_cast<const f32x4*>(&rks[16 * w + 4 * g]);
  const float Gq = G[mine];
  Parts4<2> p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    p[j] = {};
    if (j > w) continue;
    f32x4 kj_t = {}, qj_t = {};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bf16x8 kj = *reinterpret_cast<const bf16x8*>(&keys[16 * j + l16][32 * x + 8 * g]);
      kj_t = mfma16(k[x], kj, kj_t);
      qj_t = mfma16(kj, q[x], qj_t);
    }
    const float Gj = G[16 * j + l16], rj = rks[16 * j + l16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool below = j < w || 4 * g + r > l16;
      const float x = kj_t[r] * (bi[r] * rj) * __builtin_amdgcn_exp2f(Gi[r] - Gj);
      A[16 * w + 4 * g + r][16 * j + l16] = below ? x : 0.f;
    }
    const f32x4 Gk = *reinterpret_cast<const f32x4*>(&G[16 * j + 4 * g]);
    const f32x4 rk = *reinterpret_cast<const f32x4*>(&rks[16 * j + 4 * g]);
    f32x4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool seen = j < w || 4 * g + r <= l16;
      const float x = qj_t[r] * (rq * rk[r]) * __builtin_amdgcn_exp2f(Gq - Gk[r]);
      y[r] = seen ? x : 0.f;
    }
    p[j] = split4<2>(y);
  }
  // the wave's diagonal block, a column a lane (four times over), in its place
  __builtin_amdgcn_wave_barrier();
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float y = i == l16 ? 1.f : 0.f;
#pragma unroll
    for (int m = 0; m < i; ++m) y = fmaf(-A[16 * w + i][16 * w + m], x[m], y);
    x[i] = y;
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i / 4 == g) A[16 * w + i][16 * w + l16] = x[i];
  __syncthreads();
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    if (y > w / 2) continue;
    char* at = out + p_at(w, y) + 16 * lane;
#pragma unroll
    for (int z = 0; z < 2; ++z) *reinterpret_cast<u64x2*>(at + z * kFragment) = u64x2{p[2 * y].p[z], p[2 * y + 1].p[z]};
  }
  if (h == kh * group) {  // K^T: row tiles 2 w and 2 w + 1, both steps
    char* kt = work.keys + (tile * a.hk + kh) * kKeys;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int m = 2 * w + y / 2, step = y % 2;
      uint16_t e8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] = keys[32 * step + 16 * (e / 4) + 4 * g + e % 4][key_of(m, l16)];
      *reinterpret_cast<u32x4*>(kt + (2 * m + step) * kFragment + 16 * lane) = __builtin_bit_cast(u32x4, e8);
    }
  }
  // the row block, transposed: xt[j] is X_wj^T, lane: row l16 of X_wj, columns 4 g ..
  f32x4 xt[4];
  Parts4<3> px[4];
#pragma unroll
  for (int j = 3; j >= 0; --j) {
    px[j] = {};
    xt[j] = f32x4{};
    if (j > w) continue;
    if (j == w) {
      xt[j] = *reinterpret_cast<const f32x4*>(&A[16 * w + l16][16 * w + 4 * g]);
      f32x4 less = xt[j];  // the unit diagonal stays out
#pragma unroll
      for (int r = 0; r < 4; ++r) less[r] = 4 * g + r == l16 ? 0.f : less[r];
      px[j] = split4<3>(less);
      continue;
    }
    f32x4 to[3] = {};
#pragma unroll
    for (int m = 3; m > 0; --m) {
      if (m > w || m <= j) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) to[m - 1] = mfma16_f32(A[16 * m + 4 * g + r][16 * j + l16], xt[m][r], to[m - 1]);
    }
    const f32x4 all = to[0] + to[1] + to[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) xt[j] = mfma16_f32(-A[16 * j + 4 * g + r][16 * j + l16], all[r], xt[j]);
    px[j] = split4<3>(xt[j]);
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    if (y > w / 2) continue;
    char* at = out + x_at(w, y) + 16 * lane;
#pragma unroll
    for (int z = 0; z < 3; ++z) *reinterpret_cast<u64x2*>(at + z * kFragment) = u64x2{px[2 * y].p[z], px[2 * y + 1].p[z]};
  }
}

// What of the outputs is known at compile time.
enum { kAnyOut = 0, kBf16Out = 1 };

// global -> LDS, 16 bytes a lane
__device__ __forceinline__ void copy16(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
// s_waitcnt: until at most n vector-memory operations are outstanding
constexpr unsigned wait_loads(int n) { return (unsigned)((n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8)); }
// a barrier that waits for no copy
__device__ __forceinline__ void barrier_only() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr int kScanThreads = 64 * 12;

// The states through the chunks: a workgroup for 16 NT value columns of a head.
// What bounds it is the chain S -> W -> U -> S of one chunk after the other, so
// its twelve waves divide the work such that nothing else stands in it:
//   0-3  the chain: each 32 keys of S in its accumulators, as results of K^T U
//        and as terms of K S (whose four partial sums pass through the LDS), and
//        16 of the chunk's rows of W and U, which pass through the LDS as the
//        next product's operand
//   4-7  the outputs of 16 rows each, from S and U
//   8-10 copy the chain's operands to the LDS, each group as soon as the last
//        chunk's has been used (loads by the chain's waves hold them up: 64 bytes
//        a cycle and CU, 0.6 us a chunk)
//   11   reads what is needed three chunks on into the L2
// Three barriers a chunk: 1 the partial sums, 2 W, 3 U.
// The slices of a head read the same X, P, K and Q, the heads of a k head the
// same K and Q: they form a family, whose workgroups stand on one XCD, behind
// one L2 (one prompt of 8192, 16 k and 32 v heads: 2.1 GB read past the L2s with
// the slices dealt out, 0.3 so).
template <int NT, bool VEC, int OUT>
__global__ void __launch_bounds__(kScanThreads, 1) gdn_scan_kernel(const dft_prompt_gdn_args a, Work work, int families) {
  constexpr int BN = 16 * NT, kSlices = kD / BN, kSRow = kD + 8, kRow = kChunk + 8;
  __shared__ __attribute__((aligned(16))) char k_lds[16 * kFragment], kt_lds[16 * kFragment], x_lds[18 * kFragment];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[kChunk][BN];
  __shared__ __attribute__((aligned(16))) float coef_lds[2][4][kChunk];
  __shared__ __attribute__((aligned(16))) f32x4 sums[NT][4][4][64];  // [t][of wave][row tile][lane]
  __shared__ __attribute__((aligned(16))) uint16_t Sb[2][BN][kSRow];
  __shared__ __attribute__((aligned(16))) uint16_t Wb[3][BN][kRow], Ub[2][BN][kRow], Vb[3][BN][kRow];
  __shared__ __attribute__((aligned(16))) char touched[kFragment];
  if (blockIdx.x == 0 && a.status)
    for (int b = threadIdx.x; b < a.batch; b += kScanThreads)
      a.status[b] = span_of(a, b).status | slot_of(a.state_indices, a.state_indices_dtype, a.initial, a.slots, b).status;
  const int members = a.batch * a.hv / families * kSlices;  // of a family
  const int round = blockIdx.x / (kXcds * members), in = blockIdx.x - round * kXcds * members;
  const int family = round * kXcds + in % kXcds, member = in / kXcds;
  if (family >= families) return;
  const int unit = family * (members / kSlices) + member / kSlices, slice = member % kSlices, b = unit / a.hv, h = unit - b * a.hv;
  const Span s = span_of(a, b);
  if (s.n <= 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int w = wave & 3, kh = h / (a.hv / a.hk), c0 = slice * BN;
  const int64_t first = first_tile(s.r0, b, kChunk);
  const int chunks = (s.n + kChunk - 1) / kChunk;
  const uint16_t* y = static_cast<const uint16_t*>(a.y);
  auto put = [&](uint16_t* to, uint64_t x) { *reinterpret_cast<uint64_t*>(to) = x; };
  auto get = [&](const uint16_t* from) { return *reinterpret_cast<const bf16x8*>(from); };
  auto fragment = [&](const char* from) { return *reinterpret_cast<const bf16x8*>(from + 16 * lane); };
  // a row past the request's last is its last one
  auto row_at = [&](int at, int i) { return y + (s.r0 + min(at * kChunk + i, s.n - 1)) * a.y_row_stride; };
  auto head_at = [&](int at) { return work.heads + ((first + min(at, chunks - 1)) * a.hv + h) * kHead; };
  auto keys_at = [&](int at) { return work.keys + ((first + min(at, chunks - 1)) * a.hk + kh) * kKeys; };

  if (wave == 11) {
    const int part = (member % kSlices) * 64 + lane, parts = kSlices * 64;
    for (int at = 0; at < chunks; ++at) {
      if (at) {
        barrier_only();
        barrier_only();
      } else {
        barrier_only();
        barrier_only();
        barrier_only();
      }
      // lines of 128 bytes: the head's block, K^T, the rows of Q, K and V
      constexpr int kHeadLines = (kHead + 127) / 128, kKeyLines = kKeys / 128, kRowLines = 2 * kChunk;
      const int to = at + 3;
      if (to < chunks)
        for (int line = part; line < kHeadLines + kKeyLines + 3 * kRowLines; line += parts) {
          const char* from;
          int x = line;
          if (x < kHeadLines) {
            from = head_at(to) + min(x * 128, kHead - 16);
          } else if ((x -= kHeadLines) < kKeyLines) {
            from = keys_at(to) + x * 128;
          } else {
            x -= kKeyLines;
            const int which = x / kRowLines, row = x % kRowLines / 2;
            const int head = which == 0 ? kh : which == 1 ? a.hk + kh : 2 * a.hk + h;
            from = reinterpret_cast<const char*>(row_at(to, row) + head * kD) + x % 2 * 128;
          }
          copy16(from, touched);
        }
      barrier_only();
    }
    __builtin_amdgcn_s_waitcnt(wait_loads(0));
    return;
  }
  if (wave == 8) {  // X; V and the rows' factors
    auto copy_v = [&](int at) {
#pragma unroll
      for (int m = 0; m < 2 * NT; ++m)
        copy16(row_at(at, (64 * m + lane) / (2 * NT)) + (2 * a.hk + h) * kD + c0 + (64 * m + lane) % (2 * NT) * 8,
               reinterpret_cast<char*>(v_lds) + m * kFragment);
      copy16(head_at(at) + kTriangle + 16 * lane, coef_lds[at & 1]);
    };
    auto copy_x = [&](const char* head) {
#pragma unroll
      for (int m = 0; m < 18; ++m) copy16(head + m * kFragment + 16 * lane, x_lds + m * kFragment);
    };
    copy_v(0);
    copy_x(head_at(0));
    barrier_only();
    for (int at = 0; at < chunks; ++at) {
      __builtin_amdgcn_s_waitcnt(wait_loads(18));  // V
      barrier_only();                              // 1
      __builtin_amdgcn_s_waitcnt(wait_loads(0));   // X
      barrier_only();                              // 2: V has been used
      copy_v(at + 1);
      barrier_only();  // 3: X has been used
      copy_x(head_at(at + 1));
    }
    __builtin_amdgcn_s_waitcnt(wait_loads(0));
    return;
  }
  if (wave == 9) {  // K
    const uint16_t* row[4];  // rows 16 m + l16
    auto rows = [&](int at) {
#pragma unroll
      for (int m = 0; m < 4; ++m) row[m] = row_at(at, 16 * m + l16) + (a.hk + kh) * kD + 8 * g;
    };
    auto copy_k = [&]() {
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int x = 0; x < 4; ++x) copy16(row[m] + 32 * x, k_lds + (4 * x + m) * kFragment);
    };
    rows(0);
    copy_k();
    __builtin_amdgcn_s_waitcnt(wait_loads(0));
    barrier_only();
    for (int at = 0; at < chunks; ++at) {
      rows(at + 1);
      barrier_only();  // 1: K has been used
      copy_k();
      barrier_only();  // 2
      __builtin_amdgcn_s_waitcnt(wait_loads(0));
      barrier_only();  // 3
    }
    return;
  }
  if (wave == 10) {  // K^T
    barrier_only();
    for (int at = 0; at < chunks; ++at) {
      const char* keys = keys_at(at) + 16 * lane;
      barrier_only();  // 1: the last chunk's has been used
#pragma unroll
      for (int m = 0; m < 16; ++m) copy16(keys + m * kFragment, kt_lds + m * kFragment);
      barrier_only();  // 2
      __builtin_amdgcn_s_waitcnt(wait_loads(0));
      barrier_only();  // 3
    }
    return;
  }
  if (wave >= 4) {
    const bool vec = a.o_dtype == DFT_F32 && reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && a.o_row_stride % 4 == 0 && a.o_h_stride % 4 == 0;
    bf16x8 q[4], p[2][2];  // the wave's rows of Q and P
    float rq;              // e^G rq of row l16
    auto load_q = [&](int at) {
      const uint16_t* row = row_at(at, 16 * w + l16) + kh * kD + 8 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const bf16x8*>(row + 32 * j);
      rq = reinterpret_cast<const float*>(head_at(at) + kTriangle)[4 * kChunk + 16 * w + l16];
    };
    auto load_p = [&](int at) {
      const char* head = head_at(at) + 16 * lane;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          p[j][z] = *reinterpret_cast<const bf16x8*>(head + (j && w < 2 ? kTriangle + kCoef : p_at(w, j) + z * kFragment));
    };
    load_q(0);
    load_p(0);
    barrier_only();
    for (int at = 0; at < chunks; ++at) {
      f32x4 o[NT];
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 q0 = {}, q1 = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q0 = mfma16(get(&Sb[0][16 * t + l16][32 * j + 8 * g]), q[j], q0);
          q1 = mfma16(get(&Sb[1][16 * t + l16][32 * j + 8 * g]), q[j], q1);
        }
        o[t] = (q0 + q1) * rq;
      }
      load_q(at + 1);
      __syncthreads();
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 o1 = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bf16x8 u0 = get(&Ub[0][16 * t + l16][32 * j + 8 * g]);
          const bf16x8 u1 = get(&Ub[1][16 * t + l16][32 * j + 8 * g]);
          o[t] = mfma16(u0, p[j][0], o[t]);
          o1 = mfma16(u1, p[j][0], o1);
          o1 = mfma16(u0, p[j][1], o1);
        }
        o[t] += o1;
      }
      load_p(at + 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int i = at * kChunk + 16 * w + l16;
        if (i < s.n) {
          const int64_t to = (s.r0 + i) * a.o_row_stride + h * a.o_h_stride + c0 + 16 * t + 4 * g;
          if constexpr (OUT == kBf16Out) {
            typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<bf16x4*>(static_cast<uint16_t*>(a.o) + to) = __builtin_convertvector(o[t], bf16x4);
          } else if (vec) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.o) + to) = o[t];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) store(a.o, to + r, a.o_dtype, o[t][r]);
          }
        }
      }
    }
    return;
  }

  const Slot slot = slot_of(a.state_indices, a.state_indices_dtype, a.initial, a.slots, b);
  f32x4 S[2][NT];  // keys 32 w + 8 g + 4 x .., column 16 t + l16
  float* state = a.state + slot.at * a.state_slot_stride + h * a.state_h_stride;
  auto key_at = [&](int x, int t) {
    return (32 * w + 8 * g + 4 * x) * a.state_k_stride + (c0 + 16 * t + l16) * a.state_v_stride;
  };
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      S[x][t] = f32x4{};
      if (!slot.initial) continue;
      if constexpr (VEC)
        S[x][t] = *reinterpret_cast<const f32x4*>(state + key_at(x, t));
      else
#pragma unroll
        for (int r = 0; r < 4; ++r) S[x][t][r] = state[key_at(x, t) + r * a.state_k_stride];
    }
  const int place = 32 * (w / 2) + 8 * g + 4 * (w % 2);  // of the lane's rows 16 w + 4 g .. as terms
  __builtin_amdgcn_s_setprio(2);
  __syncthreads();
  for (int at = 0; at < chunks; ++at) {
    const float(*coef)[kChunk] = coef_lds[at & 1];
    f32x4 u[NT];
    bf16x8 k[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) k[m] = fragment(k_lds + (4 * w + m) * kFragment);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Parts4<3> lo = split4<3>(S[0][t]), hi = split4<3>(S[1][t]);
      bf16x8 p[3];
#pragma unroll
      for (int z = 0; z < 3; ++z) p[z] = __builtin_bit_cast(bf16x8, u64x2{lo.p[z], hi.p[z]});
      f32x4 sum[4] = {};
#pragma unroll
      for (int z = 2; z >= 0; --z)
#pragma unroll
        for (int m = 0; m < 4; ++m) sum[m] = mfma16(k[m], p[z], sum[m]);
#pragma unroll
      for (int z = 0; z < 2; ++z) *reinterpret_cast<bf16x8*>(&Sb[z][16 * t + l16][32 * w + 8 * g]) = p[z];
#pragma unroll
      for (int m = 0; m < 4; ++m) sums[t][w][m][lane] = sum[m];
    }
    __syncthreads();
    const f32x4 beta = *reinterpret_cast<const f32x4*>(&coef[0][16 * w + 4 * g]);
    const f32x4 decayed = *reinterpret_cast<const f32x4*>(&coef[1][16 * w + 4 * g]);
    const f32x4 out = *reinterpret_cast<const f32x4*>(&coef[2][16 * w + 4 * g]);
    const float keep = coef[3][0];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const f32x4 ks = (sums[t][0][w][lane] + sums[t][1][w][lane]) + (sums[t][2][w][lane] + sums[t][3][w][lane]);
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = bf16_bits_to_f32(v_lds[16 * w + 4 * g + r][16 * t + l16]);
      u[t] = beta * v - decayed * ks;
      const Parts4<3> p = split4<3>(u[t]);
#pragma unroll
      for (int z = 0; z < 3; ++z) put(&Wb[z][16 * t + l16][place], p.p[z]);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x4 u1 = {}, u2 = {};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j > w / 2) continue;
        const bf16x8 w0 = get(&Wb[0][16 * t + l16][32 * j + 8 * g]);
        const bf16x8 w1 = get(&Wb[1][16 * t + l16][32 * j + 8 * g]);
        const bf16x8 w2 = get(&Wb[2][16 * t + l16][32 * j + 8 * g]);
        const char* at = x_lds + x_at(w, j);
        const bf16x8 x0 = fragment(at), x1 = fragment(at + kFragment), x2 = fragment(at + 2 * kFragment);
        u1 = mfma16(x0, w0, u1);
        u2 = mfma16(x1, w0, u2);
        u1 = mfma16(x0, w1, u1);
        u2 = mfma16(x2, w0, u2);
        u1 = mfma16(x0, w2, u1);
        u2 = mfma16(x1, w1, u2);
      }
      u[t] += u1 + u2;
      const Parts4<3> d = split4<3>(u[t] * out);
#pragma unroll
      for (int z = 0; z < 3; ++z) put(&Vb[z][16 * t + l16][place], d.p[z]);
      const Parts4<2> p = split4<2>(u[t]);
#pragma unroll
      for (int z = 0; z < 2; ++z) put(&Ub[z][16 * t + l16][place], p.p[z]);
    }
    __syncthreads();
    bf16x8 kt[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j) kt[x][j] = fragment(kt_lds + (2 * (2 * w + x) + j) * kFragment);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x4 add[2] = {};
#pragma unroll
      for (int x = 0; x < 2; ++x) S[x][t] *= keep;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bf16x8 d0 = get(&Vb[0][16 * t + l16][32 * j + 8 * g]);
        const bf16x8 d1 = get(&Vb[1][16 * t + l16][32 * j + 8 * g]);
        const bf16x8 d2 = get(&Vb[2][16 * t + l16][32 * j + 8 * g]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          S[x][t] = mfma16(kt[x][j], d0, S[x][t]);
          add[x] = mfma16(kt[x][j], d1, add[x]);
          add[x] = mfma16(kt[x][j], d2, add[x]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) S[x][t] += add[x];
    }
  }
  if (slot.at < 0) return;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (VEC)
        *reinterpret_cast<f32x4*>(state + key_at(x, t)) = S[x][t];
      else
#pragma unroll
        for (int r = 0; r < 4; ++r) state[key_at(x, t) + r * a.state_k_stride] = S[x][t][r];
    }
}

// Whether a state's columns are read in 16-byte pieces.
bool vector_state(const dft_prompt_gdn_args& a) {
  return a.state_k_stride == 1 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0 && a.state_v_stride % 4 == 0 &&
         a.state_h_stride % 4 == 0 && a.state_slot_stride % 4 == 0;
}

bool by_rows(const dft_prompt_gdn_args& a) { return a.max_len <= 2; }
int64_t tiles_of(const dft_prompt_gdn_args& a) { return line_tiles(a.rows, a.batch, kChunk); }

template <int NT>
int launch_scan(const dft_prompt_gdn_args& a, const Work& work, hipStream_t stream) {
  // by k heads where there is one for every XCD, else by v heads
  const int families = a.batch * (a.batch * a.hk >= kXcds ? a.hk : a.hv);
  const unsigned blocks = (unsigned)((families + kXcds - 1) / kXcds * kXcds * (a.batch * a.hv / families * (8 / NT)));
  const bool bf16 = a.o_dtype == DFT_BF16 && reinterpret_cast<uintptr_t>(a.o) % 8 == 0 && a.o_row_stride % 4 == 0 && a.o_h_stride % 4 == 0;
  if (!vector_state(a))
    gdn_scan_kernel<NT, false, kAnyOut><<<blocks, kScanThreads, 0, stream>>>(a, work, families);
  else if (bf16)
    gdn_scan_kernel<NT, true, kBf16Out><<<blocks, kScanThreads, 0, stream>>>(a, work, families);
  else
    gdn_scan_kernel<NT, true, kAnyOut><<<blocks, kScanThreads, 0, stream>>>(a, work, families);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace

// the most workgroups of a launch
int64_t prompt_gdn_blocks(const dft_prompt_gdn_args* a) {
  return std::max(((int64_t)a->batch * a->hv + kXcds * a->hv) * 8 * 2, by_rows(*a) ? 0 : tiles_of(*a) * a->hv);
}
int64_t prompt_gdn_workspace(const dft_prompt_gdn_args* a) {
  return by_rows(*a) ? 0 : tiles_of(*a) * ((int64_t)a->hv * kHead + (int64_t)a->hk * kKeys);
}

int launch_prompt_gdn(const dft_prompt_gdn_args* a, hipStream_t stream) {
  if (by_rows(*a)) {
    const unsigned blocks = (unsigned)((int64_t)a->batch * a->hv);
    if (vector_state(*a))
      gdn_rows_kernel<128, true><<<blocks, 256, 0, stream>>>(*a);
    else
      gdn_rows_kernel<128, false><<<blocks, 256, 0, stream>>>(*a);
    return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
  }
  Work work;
  work.heads = static_cast<char*>(a->workspace);
  work.keys = work.heads + tiles_of(*a) * a->hv * kHead;
  gdn_chunk_kernel<<<(unsigned)(tiles_of(*a) * a->hv), 256, 0, stream>>>(*a, work);
  if (hipGetLastError() != hipSuccess) return DFT_ERR_LAUNCH;
  return launch_scan<1>(*a, work, stream);
}

}  // namespace dft
