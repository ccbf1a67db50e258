// dft_prompt_gdn: the gated delta rule over packed prompts and single tokens.
//
// Per v head and row, q and k normalised, q scaled:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q
// Single tokens: row by row, gdn_rows_kernel.  Prompts: in chunks of 64 rows,
// for whose rows i and j, G the running sum of g within the chunk, K and Q the
// raw rows, rk and rq what normalises (and scales) them:
//   A_ij = beta_i rk_i rk_j (k_i . k_j) e^(G_i - G_j)  (j < i),  X = (I + A)^-1
//   W = beta (V - e^G rk (K S)),  U = rk (X W)
//   O = rq (e^G (Q S) + P U),  P_ij = (q_i . k_j) e^(G_i - G_j)  (j <= i)
//   S <- e^G_63 S + K^T (e^(G_63 - G) U)
// gdn_chunk_kernel forms what needs no state, X and P, for all chunks at once,
// gdn_scan_kernel takes the states through the chunks.  The raw rows are bf16,
// so that K, Q and K^T are exact operands of bf16 products.  What is not goes in
// as a sum of three bf16 parts, 2^-24 relative at most, and a product of two such
// factors as its six of 2^-16 or more.  (With two parts states and fp32 outputs
// come out 4 10^-6 off.  Two where only outputs pass through: 6 to 10% less time.)
#include <algorithm>
#include <type_traits>

#include "packed.h"

namespace dft {
namespace {

using namespace packed;

constexpr int kD = 128;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// g and beta of one row and head
struct Gate {
  float g, beta;
};
struct GateOf {  // of a head
  float rate, bias;
  __device__ __forceinline__ GateOf(const dft_prompt_gdn_args& a, int h)
      : rate(a.neg_exp_A ? a.neg_exp_A[h] : -expf(ld_f(a.A_log, h, a.A_log_dtype))), bias(ld_f(a.dt_bias, h, a.dt_bias_dtype)) {}
  __device__ __forceinline__ Gate operator()(float a, float b) const {
    const float x = a + bias, soft = x > 20.f ? x : log1pf(expf(x));
    return {rate * soft, 1.f / (1.f + expf(-b))};
  }
};
__device__ __forceinline__ float gate_a(const dft_prompt_gdn_args& a, int64_t row, int h) { return ld_f(a.a, row * a.a_row_stride + h, a.a_dtype); }
__device__ __forceinline__ float gate_b(const dft_prompt_gdn_args& a, int64_t row, int h) { return ld_f(a.b, row * a.b_row_stride + h, a.b_dtype); }

// The sum over a row of 16 lanes, in all of them: rotations by 8, 4, 2 and 1
// within the row.
__device__ __forceinline__ float sum16(float x) {
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x128, 0xf, 0xf, true));
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x124, 0xf, 0xf, true));
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x122, 0xf, 0xf, true));
  x += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x121, 0xf, 0xf, true));
  return x;
}

// ---- row by row ------------------------------------------------------------
// A workgroup of four waves keeps V value columns of one head's state in
// registers: 16 lanes a column, 8 keys a lane (4 i .. and 64 + 4 i ..), so that
// a wave's access covers whole columns and both sums over the keys stay within
// 16 lanes.  Bound by the states' bytes: 64 requests of 32 heads 50.8 us, 5.3
// TB/s (written past the caches; through them 62.5.  Half the columns a
// workgroup 60.7, a quarter 68).  A pool whose values lie side by side is read and
// written by elements: 143.
template <int V, bool VEC>
__global__ void __launch_bounds__(256) gdn_rows_kernel(const dft_prompt_gdn_args a, int most) {
  constexpr int kSplit = kD / V, kPass = V / 16;
  const int64_t x = blockIdx.x;
  if (x == 0 && a.status)
    for (int b = threadIdx.x; b < a.batch; b += 256)
      a.status[b] = span_of(a, b).status | slot_of(a.state_indices, a.state_indices_dtype, a.initial, a.slots, b).status;
  const int per = a.hv * kSplit;
  const int b = (int)(x / per), in = (int)(x - (int64_t)b * per), h = in / kSplit, part = in - h * kSplit;
  const Span s = span_of(a, b);
  if (s.n <= 0 || s.n > most) return;
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
  // a row's inputs, fetched a row ahead
  struct Row {
    u32x2 q[2], k[2];
    uint16_t v[kPass];
    float a, b;
  };
  const uint16_t* y = static_cast<const uint16_t*>(a.y) + s.r0 * a.y_row_stride;
  auto fetch = [&](Row& r, int t) {
    const uint16_t* yr = y + t * a.y_row_stride;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      r.q[x] = *reinterpret_cast<const u32x2*>(yr + kh * kD + 4 * i + 64 * x);
      r.k[x] = *reinterpret_cast<const u32x2*>(yr + (a.hk + kh) * kD + 4 * i + 64 * x);
    }
#pragma unroll
    for (int p = 0; p < kPass; ++p) r.v[p] = yr[(2 * a.hk + h) * kD + v0 + 4 * p];
    r.a = gate_a(a, s.r0 + t, h);
    r.b = gate_b(a, s.r0 + t, h);
  };
  const GateOf gate(a, h);
  Row r;
  fetch(r, 0);
  for (int t = 0; t < s.n; ++t) {
    Row next = r;
    if (t + 1 < s.n) fetch(next, t + 1);
    float q[8], k[8], qq = 0, kk = 0, qk = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] = bf16_bits_to_f32(r.q[e >> 2][e >> 1 & 1] >> (e & 1) * 16);
      k[e] = bf16_bits_to_f32(r.k[e >> 2][e >> 1 & 1] >> (e & 1) * 16);
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
    const Gate g = gate(r.a, r.b);
    const float decay = expf(g.g);
    float out = 0;
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
      const float u = g.beta * (bf16_bits_to_f32(r.v[p]) - kS);
#pragma unroll
      for (int e = 0; e < 8; ++e) S[p][e] = fmaf(k[e], u, S[p][e]);
      if (i == p) out = fmaf(qk, u, qS);
    }
    if (i < kPass) store(a.o, (s.r0 + t) * a.o_row_stride + h * a.o_h_stride + v0 + 4 * i, a.o_dtype, out);
    r = next;
  }
  if (slot.at < 0) return;
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    if constexpr (VEC) {
#pragma unroll
      for (int y = 0; y < 2; ++y)
        __builtin_nontemporal_store(f32x4{S[p][4 * y], S[p][4 * y + 1], S[p][4 * y + 2], S[p][4 * y + 3]},
                                    reinterpret_cast<f32x4*>(state + at(p, 4 * y)));
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
constexpr int kChunk = 64, kXcds = 8, kCus = 256;
constexpr int kFragment = 1024;  // bytes: 64 lanes x 16
// X - I, whose upper half is zero, in fp32: its row tile m (of 16) has steps 0 ..
// m / 2, six fragments of 8 elements a lane, the first four of every lane first.
constexpr int kX = 6 * 2 * kFragment;
__host__ __device__ constexpr int x_at(int m, int s) { return m < 2 ? m : 2 * m - 2 + s; }
// P's six in three parts, and a fragment of zeros for the other step of the row
// tiles 0 and 1, so that all waves do the same (loads whose use depends on the
// wave are waited for too early).
constexpr int kP = (6 * 3 + 1) * kFragment;
__host__ __device__ constexpr int p_at(int m, int s) { return m < 2 && s ? 18 : 3 * x_at(m, s); }
// Factors of the rows, 64 floats each: beta, e^G rk beta, rk, e^(G_63 - G), e^G_63 (of all); e^G, rq.
enum { kBeta, kDecayed, kUnit, kOut, kKeep, kDecay, kRq, kCoefs = 8 };
constexpr int kHead = kX + kP + kCoefs * kChunk * 4;

struct Work {
  char* heads;  // [tile][hv][kHead]: X - I in fp32, P, the rows' factors
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

// A row's decay, in log2 units, down to which it matters: 2^-512 is zero in fp32
// already, for this row and for every span of rows that it is one of, and sums
// stay finite.
constexpr double kLeast = -512;

// X and P of a chunk and v head: a workgroup of four waves, wave w for rows 16 w ...
// Row block by row block from X (I + A) = I: diagonal blocks by substitution
// (their powers would lose what equal keys leave of 32 bits), then X_ij =
// -(sum_(j<m<=i) X_im A_mj) X_jj in fp32 products, transposed, so that each result
// is the next one's operand and the last the fragment that is stored.
// A decay between two rows is the difference of two running sums: they are added
// up in 64 bits and kept in two floats, or a few rows that leave nothing of the
// state would leave the weak gates behind them a sum of thousands, in steps of
// 10^-3 (24 rows of g = -300 among weak ones: states 4 10^-4 off, so 1 10^-7).
// Bound by the instructions that its waves issue, so by what of them stand ready:
// 128 registers, four workgroups a CU.  A prompt of 8192 rows and 32 heads 54 us
// for 213 MB read and written, 4.0 TB/s; with two workgroups a CU, and two parts
// of P, 78 where it took 52.
__global__ void __launch_bounds__(256, 4) gdn_chunk_kernel(const dft_prompt_gdn_args a, Work work, int past) {
  constexpr int kKRow = kD + 8, kARow = kChunk + 4;
  __shared__ __attribute__((aligned(16))) uint16_t keys[kChunk][kKRow];
  __shared__ __attribute__((aligned(16))) float A[kChunk][kARow];
  __shared__ __attribute__((aligned(16))) float G[2][kChunk], beta[kChunk], rks[kChunk];
  // the v heads of a k head read the same rows: one after the other on one XCD
  const int share = a.hv / a.hk, in = blockIdx.x / kXcds;
  const int64_t unit = (int64_t)(in / share) * kXcds + blockIdx.x % kXcds, tile = unit / a.hk;
  const int kh = (int)(unit - tile * a.hk), h = kh * share + in % share;
  const int b = find_tile<256>(a, tile, kChunk);
  if (b < 0) return;
  const Span s = span_of(a, b);
  if (s.n <= past) return;
  const int t0 = (int)(tile - first_tile(s.r0, b, kChunk)) * kChunk, n = min(s.n - t0, kChunk);
  const int64_t r0 = s.r0 + t0;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;

  // rows past the request's last: zeros
  const int mine = 16 * w + l16;
  const uint16_t* row = static_cast<const uint16_t*>(a.y) + (r0 + min(mine, n - 1)) * a.y_row_stride + (a.hk + kh) * kD + 8 * g;
  u32x4 kw[4], qw[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) kw[j] = *reinterpret_cast<const u32x4*>(row + 32 * j);
#pragma unroll
  for (int j = 0; j < 4; ++j) qw[j] = *reinterpret_cast<const u32x4*>(row - a.hk * kD + 32 * j);
  Gate gate = {};
  double sum = 0, all = 0;
  if (w == 0) {  // the gates, a row a lane, G in log2 units
    const int64_t r = r0 + min(lane, n - 1);
    gate = GateOf(a, h)(gate_a(a, r, h), gate_b(a, r, h));
    if (lane >= n) gate.g = gate.beta = 0;
    sum = gate.g * 1.4426950408889634;
    if (sum < kLeast) sum = kLeast;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(sum, o);
      if (lane >= o) sum += up;
    }
    all = __shfl(sum, 63);
    G[0][lane] = (float)sum;
    G[1][lane] = (float)(sum - (float)sum);
    beta[lane] = gate.beta;
  }
  // the norms stand on the diagonals of the wave's own Gram tiles: row l16's in lane (l16, l16 / 4), register l16 % 4
  bf16x8 k[4], q[4];
  f32x4 kk = {}, qq = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (mine >= n) kw[j] = qw[j] = u32x4{};
    k[j] = __builtin_bit_cast(bf16x8, kw[j]);
    q[j] = __builtin_bit_cast(bf16x8, qw[j]);
    *reinterpret_cast<u32x4*>(&keys[mine][32 * j + 8 * g]) = kw[j];
    kk = mfma16(k[j], k[j], kk);
    qq = mfma16(q[j], q[j], qq);
  }
  char* out = work.heads + (tile * a.hv + h) * kHead;
  if (l16 / 4 == g) {
    auto own = [&](f32x4 x) { return l16 & 2 ? (l16 & 1 ? x[3] : x[2]) : (l16 & 1 ? x[1] : x[0]); };
    rks[mine] = 1.f / sqrtf(own(kk) + 1e-6f);
    reinterpret_cast<float*>(out + kX + kP)[kRq * kChunk + mine] = a.scale / sqrtf(own(qq) + 1e-6f);
  }
  __syncthreads();

  if (w == 0) {
    float* coef = reinterpret_cast<float*>(out + kX + kP) + lane;
    const float rk = rks[lane];
    coef[kBeta * kChunk] = gate.beta;
    const float decay = __builtin_amdgcn_exp2f((float)sum);
    coef[kDecayed * kChunk] = lane < n ? decay * rk * gate.beta : 0;
    coef[kUnit * kChunk] = lane < n ? rk : 0;
    coef[kOut * kChunk] = lane < n ? __builtin_amdgcn_exp2f((float)(all - sum)) : 0;
    coef[kKeep * kChunk] = __builtin_amdgcn_exp2f((float)all);
    coef[kDecay * kChunk] = decay;
    *reinterpret_cast<u32x4*>(out + kX + 18 * kFragment + 16 * lane) = u32x4{};
  }

  // A into the LDS, P to its place, transposed: Gram tiles K K^T and K Q^T of the keys of tiles j <= w with the wave's rows
  const float Gq = G[0][mine], Gq_low = G[1][mine], bk = beta[mine] * rks[mine];
  Parts4<3> p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    p[j] = {};
    if (j > w) continue;
    f32x4 dot = {}, qk = {};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bf16x8 kj = *reinterpret_cast<const bf16x8*>(&keys[16 * j + l16][32 * x + 8 * g]);
      dot = mfma16(kj, k[x], dot);
      qk = mfma16(kj, q[x], qk);
    }
    const f32x4 Gk = *reinterpret_cast<const f32x4*>(&G[0][16 * j + 4 * g]);
    const f32x4 Gk_low = *reinterpret_cast<const f32x4*>(&G[1][16 * j + 4 * g]);
    const f32x4 rk = *reinterpret_cast<const f32x4*>(&rks[16 * j + 4 * g]);
    f32x4 x, y;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ahead = j < w ? 1 : l16 - (4 * g + r);  // of the key the row is
      const float decay = __builtin_amdgcn_exp2f((Gq - Gk[r]) + (Gq_low - Gk_low[r]));
      x[r] = ahead > 0 ? dot[r] * (bk * rk[r]) * decay : 0.f;
      y[r] = ahead >= 0 ? qk[r] * decay : 0.f;
    }
    *reinterpret_cast<f32x4*>(&A[mine][16 * j + 4 * g]) = x;
    p[j] = split4<3>(y);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (j > w / 2) continue;
#pragma unroll
    for (int z = 0; z < 3; ++z)
      *reinterpret_cast<u64x2*>(out + kX + (p_at(w, j) + z) * kFragment + 16 * lane) = u64x2{p[2 * j].p[z], p[2 * j + 1].p[z]};
  }
  // the wave's diagonal block: its two halves' inverses D by substitution, a column a lane (four times over), and with L
  // what is below them X = D - D L D
  __builtin_amdgcn_wave_barrier();
  f32x4 diagonal;
  {
    const int at = 16 * w + (l16 & 8);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float y = i == (l16 & 7) ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) y = fmaf(-A[at + i][at + m], x[m], y);
      x[i] = y;
    }
    __builtin_amdgcn_wave_barrier();
    if (g == 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) A[at + i][16 * w + l16] = x[i];
    __builtin_amdgcn_wave_barrier();
    diagonal = *reinterpret_cast<const f32x4*>(&A[mine][16 * w + 4 * g]);
    if (l16 >= 8 && g < 2) diagonal = f32x4{};
    const bool below = g >= 2 && l16 < 8;
    float D[4];
    f32x4 DL = {};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float y = A[16 * w + 4 * g + r][16 * w + l16];
      D[r] = below ? 0.f : -y;
      DL = mfma16_f32(below ? y : 0.f, diagonal[r], DL);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) diagonal = mfma16_f32(D[r], DL[r], diagonal);
    __builtin_amdgcn_wave_barrier();
    *reinterpret_cast<f32x4*>(&A[mine][16 * w + 4 * g]) = diagonal;
  }
  __syncthreads();
  // the row block, transposed: xt[j] is X_wj^T, lane: row l16 of X_wj, columns 4 g ..
  auto row_block = [&](auto which) {
    constexpr int W = decltype(which)::value;
    f32x4 xt[4] = {};
    xt[W] = diagonal;
#pragma unroll
    for (int j = W - 1; j >= 0; --j) {
      f32x4 to[3] = {}, all = {};
#pragma unroll
      for (int m = W; m > j; --m)
#pragma unroll
        for (int r = 0; r < 4; ++r) to[m - 1] = mfma16_f32(A[16 * m + 4 * g + r][16 * j + l16], xt[m][r], to[m - 1]);
#pragma unroll
      for (int m = W; m > j; --m) all += to[m - 1];
#pragma unroll
      for (int r = 0; r < 4; ++r) xt[j] = mfma16_f32(-A[16 * j + 4 * g + r][16 * j + l16], all[r], xt[j]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) xt[W][r] = 4 * g + r == l16 ? 0.f : xt[W][r];  // the unit diagonal stays out
#pragma unroll
    for (int j = 0; j < 2 * (W / 2) + 2; ++j)
      *reinterpret_cast<f32x4*>(out + (2 * x_at(W, j / 2) + j % 2) * kFragment + 16 * lane) = xt[j];
  };
  switch (w) {
    case 0: return row_block(std::integral_constant<int, 0>());
    case 1: return row_block(std::integral_constant<int, 1>());
    case 2: return row_block(std::integral_constant<int, 2>());
    default: return row_block(std::integral_constant<int, 3>());
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

// The request at this place in the order of falling lengths, of at most 64: the
// others as they come.  (20 prompts of 500 rows and one of 8192 behind them: 600
// us, as they come 733; six of 257 to 2999 no better for it.)
__device__ __forceinline__ int nth_longest(const dft_prompt_gdn_args& a, int place) {
  if (!a.cu_seqlens || a.batch == 1 || a.batch > 64) return place;
  const int lane = threadIdx.x & 63, n = lane < a.batch ? span_of(a, lane).n : 0;
  int longer = 0;
  for (int i = 0; i < a.batch; ++i) {
    const int other = __builtin_amdgcn_readlane(n, i);
    longer += other > n || (other == n && i < lane);
  }
  return __ffsll((unsigned long long)__ballot(lane < a.batch && longer == place)) - 1;
}

// The states through the chunks: a workgroup for 16 NT value columns of a head.
// What bounds it is the chain S -> W -> U -> S of one chunk after the other, and
// beside it the bytes that a CU gets from its L2 (some 23 a cycle).  So its
// twelve waves divide the work such that nothing else stands in the chain, and
// K is read once for K S and K^T U:
//   0-3   the chain: each 32 keys of S in its accumulators, as results of K^T U
//         and as terms of K S (whose four partial sums pass through the LDS), and
//         16 of the chunk's rows of W and U, which pass through the LDS as the
//         next product's operand
//   4-7   the outputs of 16 rows each, from S and U
//   8     copies K, V and the rows' factors to the LDS (loads by the chain's
//         waves would hold them up)
//   9-11  split X
// Three barriers a chunk: 1 the partial sums, 2 W, 3 U.
// The slices of a head read the same X, K and Q, the heads of a k head the same
// K and Q: they form a family, whose workgroups stand on one XCD, behind one L2
// (a prompt of 8192 rows, 16 k and 32 v heads: 2.1 GB read past the L2s with the
// slices dealt out, 0.3 so).  That prompt's states take 217 us, 1.7 a chunk (237
// under the profiler): the matrix unit is busy 24% of it and the LDS 56, the waves wait 55%.
template <int NT, bool VEC, int OUT>
__global__ void __launch_bounds__(kScanThreads, 1) gdn_scan_kernel(const dft_prompt_gdn_args a, Work work, int families, int past) {
  constexpr int BN = 16 * NT, kSlices = kD / BN, kSRow = kD + 8, kRow = kChunk + 8;
  // K's fragments (step x, row tile m) at 4 x + m; what lane (row l16, terms 8 g ..) takes lies in its place key_place
  __shared__ __attribute__((aligned(16))) char k_lds[2][16 * kFragment], x_lds[18 * kFragment];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[kChunk][BN];
  __shared__ __attribute__((aligned(16))) float coef_lds[2][kCoefs][kChunk];
  __shared__ __attribute__((aligned(16))) f32x4 sums[NT][4][4][64];  // [t][of wave][row tile][lane]
  __shared__ __attribute__((aligned(16))) uint16_t Sb[3][BN][kSRow];
  __shared__ __attribute__((aligned(16))) uint16_t Wb[3][BN][kRow], Ub[3][BN][kRow], Vb[3][BN][kRow];
  if (blockIdx.x == 0 && a.status)
    for (int b = threadIdx.x; b < a.batch; b += kScanThreads)
      a.status[b] = span_of(a, b).status | slot_of(a.state_indices, a.state_indices_dtype, a.initial, a.slots, b).status;
  const int members = a.batch * a.hv / families * kSlices;  // of a family
  const int round = blockIdx.x / (kXcds * members), in = blockIdx.x - round * kXcds * members;
  const int family = round * kXcds + in % kXcds, member = in / kXcds;
  if (family >= families) return;
  const int unit = family * (members / kSlices) + member / kSlices, slice = member % kSlices;
  const int turn = unit / a.hv, h = unit - turn * a.hv, b = nth_longest(a, turn);
  const Span s = span_of(a, b);
  if (s.n <= past) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int w = wave & 3, kh = h / (a.hv / a.hk), c0 = slice * BN;
  const int64_t first = first_tile(s.r0, b, kChunk);
  const int chunks = (s.n + kChunk - 1) / kChunk;
  const uint16_t* y = static_cast<const uint16_t*>(a.y);
  auto put = [&](uint16_t* to, uint64_t x) { *reinterpret_cast<uint64_t*>(to) = x; };
  auto get = [&](const uint16_t* from) { return *reinterpret_cast<const bf16x8*>(from); };
  // where row i of a row tile has its terms 8 c ..: no two of 16 lanes that read side by side share a bank
  auto key_place = [](int i, int c) { return 64 * i + 16 * (c ^ (i >> 2 & 3)); };
  // a row past the request's last is its last one
  auto row_at = [&](int at, int i) { return y + (s.r0 + min(at * kChunk + i, s.n - 1)) * a.y_row_stride; };
  auto head_at = [&](int at) { return work.heads + ((first + min(at, chunks - 1)) * a.hv + h) * kHead; };

  if (wave >= 9) {
    const int x0 = 2 * (wave - 9);  // the wave's two fragments
    f32x4 from[2][2];
    auto load_x = [&](int at) {
      const char* head = head_at(at) + 16 * lane;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 2; ++j) from[x][j] = *reinterpret_cast<const f32x4*>(head + (2 * (x0 + x) + j) * kFragment);
    };
    u64x2 to[2][3];
    auto split = [&]() {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const Parts4<3> lo = split4<3>(from[x][0]), hi = split4<3>(from[x][1]);
#pragma unroll
        for (int z = 0; z < 3; ++z) {
          to[x][z] = u64x2{lo.p[z], hi.p[z]};
          asm volatile("" : "+v"(to[x][z]));  // here, not behind the barrier
        }
      }
    };
    auto write = [&]() {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int z = 0; z < 3; ++z) *reinterpret_cast<u64x2*>(x_lds + (3 * (x0 + x) + z) * kFragment + 16 * lane) = to[x][z];
    };
    load_x(0);
    split();
    write();
    load_x(1);
    barrier_only();
    for (int at = 0; at < chunks; ++at) {
      __syncthreads();  // 1
      split();
      barrier_only();  // 2: X has been read
      write();
      load_x(at + 2);
      barrier_only();  // 3
    }
    return;
  }
  if (wave == 8) {
    const int i = lane >> 2, c = (lane & 3) ^ (i >> 2 & 3);  // key_place
    const uint16_t *k_row[4], *v_row[2 * NT];
    const char* coef;
    auto find_k = [&](int at) {
#pragma unroll
      for (int m = 0; m < 4; ++m) k_row[m] = row_at(at, 16 * m + i) + (a.hk + kh) * kD + 8 * c;
    };
    auto find_v = [&](int at) {
#pragma unroll
      for (int m = 0; m < 2 * NT; ++m)
        v_row[m] = row_at(at, (64 * m + lane) / (2 * NT)) + (2 * a.hk + h) * kD + c0 + (64 * m + lane) % (2 * NT) * 8;
      coef = head_at(at) + kX + kP + 16 * lane;
    };
    auto copy_k = [&](int at) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int x = 0; x < 4; ++x) copy16(k_row[m] + 32 * x, k_lds[at & 1] + (4 * x + m) * kFragment);
    };
    auto copy_v = [&](int at) {
#pragma unroll
      for (int m = 0; m < 2 * NT; ++m) copy16(v_row[m], reinterpret_cast<char*>(v_lds) + m * kFragment);
#pragma unroll
      for (int m = 0; m < 2; ++m) copy16(coef + m * kFragment, reinterpret_cast<char*>(coef_lds[at & 1]) + m * kFragment);
    };
    find_k(0);
    find_v(0);
    copy_k(0);
    copy_v(0);
    find_k(1);
    copy_k(1);
    __builtin_amdgcn_s_waitcnt(wait_loads(16));
    barrier_only();
    for (int at = 0; at < chunks; ++at) {
      __builtin_amdgcn_s_waitcnt(wait_loads(16));  // V
      barrier_only();                              // 1
      find_v(at + 1);
      find_k(at + 2);
#pragma unroll
      for (int m = 0; m < 4; ++m) asm volatile("" : "+v"(k_row[m]));  // here, not behind the barriers
#pragma unroll
      for (int m = 0; m < 2 * NT; ++m) asm volatile("" : "+v"(v_row[m]));
      barrier_only();  // 2: V has been read
      copy_v(at + 1);
      __builtin_amdgcn_s_waitcnt(wait_loads(2 * NT + 2));  // the next K
      barrier_only();                                      // 3: K has been read
      copy_k(at + 2);
    }
    __builtin_amdgcn_s_waitcnt(wait_loads(0));
    return;
  }
  if (wave >= 4) {
    const bool vec = a.o_dtype == DFT_F32 && reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && a.o_row_stride % 4 == 0 && a.o_h_stride % 4 == 0;
    bf16x8 q[4], p[2][3];  // the wave's rows of Q and P
    float decay, rq;       // of row l16
    auto load_q = [&](int at) {
      const uint16_t* row = row_at(at, 16 * w + l16) + kh * kD + 8 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const bf16x8*>(row + 32 * j);
    };
    auto load_p = [&](int at) {
      const char* head = head_at(at) + kX;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int z = 0; z < 3; ++z)
          p[j][z] = *reinterpret_cast<const bf16x8*>(head + (p_at(w, j) + (j && w < 2 ? 0 : z)) * kFragment + 16 * lane);
      const float* coef = reinterpret_cast<const float*>(head + kP) + 16 * w + l16;
      decay = coef[kDecay * kChunk];
      rq = coef[kRq * kChunk];
    };
    int64_t o_at = (s.r0 + 16 * w + l16) * a.o_row_stride + h * a.o_h_stride + c0 + 4 * g;
    load_q(0);
    load_p(0);
    barrier_only();
    f32x4 o[NT];
    auto store_rows = [&](int at) {
      if (at * kChunk + 16 * w + l16 < s.n) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int64_t to = o_at + 16 * t;
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
      o_at += kChunk * a.o_row_stride;
    };
    // between barriers 3 and 1, which the chain passes fastest, only the products
    for (int at = 0; at < chunks; ++at) {
      __syncthreads();  // 1: S is there
      if (at) {
        store_rows(at - 1);
        load_p(at);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 sum[3] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int z = 0; z < 3; ++z) sum[z] = mfma16(get(&Sb[z][16 * t + l16][32 * j + 8 * g]), q[j], sum[z]);
        o[t] = (sum[0] + (sum[1] + sum[2])) * decay;
      }
      load_q(at + 1);
      __syncthreads();  // 2
      __syncthreads();  // 3: U is there
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 o0 = o[t], o1 = {}, o2 = {}, o3 = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          bf16x8 u[3];
#pragma unroll
          for (int z = 0; z < 3; ++z) u[z] = get(&Ub[z][16 * t + l16][32 * j + 8 * g]);
          o0 = mfma16(u[0], p[j][0], o0);
          o1 = mfma16(u[1], p[j][0], o1);
          o2 = mfma16(u[0], p[j][1], o2);
          o3 = mfma16(u[1], p[j][1], o3);
          o1 = mfma16(u[2], p[j][0], o1);
          o2 = mfma16(u[0], p[j][2], o2);
        }
        o[t] = (o0 + ((o1 + o2) + o3)) * rq;
      }
    }
    store_rows(chunks - 1);
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
  // K^T: row tile x of the wave's keys, terms of step j.  A transposing read hands 16 lanes' pieces of 4 keys (piece lane %
  // 4) in 4 rows (lane / 4 % 4) out by the keys: lane l16 gets key 32 w + 8 (l16 / 4) + 4 x + l16 % 4.
  auto transposed = [&](const char* keys, int x, int j) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* Lds;
    const int at = key_place(4 * g + (l16 >> 2), lane & 3) + 8 * x;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(keys + 2 * j * kFragment + at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(keys + (2 * j + 1) * kFragment + at));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  __builtin_amdgcn_s_setprio(2);
  __syncthreads();
  for (int at = 0; at < chunks; ++at) {
    const float(*coef)[kChunk] = coef_lds[at & 1];
    const char* keys = k_lds[at & 1] + 4 * w * kFragment;
    f32x4 u[NT];
    bf16x8 k[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) k[m] = *reinterpret_cast<const bf16x8*>(keys + m * kFragment + key_place(l16, g));
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
      for (int z = 0; z < 3; ++z) *reinterpret_cast<bf16x8*>(&Sb[z][16 * t + l16][32 * w + 8 * g]) = p[z];
#pragma unroll
      for (int m = 0; m < 4; ++m) sums[t][w][m][lane] = sum[m];
    }
    __syncthreads();  // 1
    const f32x4 beta = *reinterpret_cast<const f32x4*>(&coef[kBeta][16 * w + 4 * g]);
    const f32x4 decayed = *reinterpret_cast<const f32x4*>(&coef[kDecayed][16 * w + 4 * g]);
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
    // what the next products take beside W and U
    bf16x8 X[2][3], kt[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int z = 0; z < 3; ++z)
        X[j][z] = *reinterpret_cast<const bf16x8*>(x_lds + (3 * x_at(w, min(j, w / 2)) + z) * kFragment + 16 * lane);
    const f32x4 unit = *reinterpret_cast<const f32x4*>(&coef[kUnit][16 * w + 4 * g]);
    const f32x4 out = *reinterpret_cast<const f32x4*>(&coef[kOut][16 * w + 4 * g]);
    const float keep = coef[kKeep][0];
    __syncthreads();  // 2
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j) kt[x][j] = transposed(keys, x, j);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x4 u1 = {}, u2 = {};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j > w / 2) continue;
        const bf16x8 w0 = get(&Wb[0][16 * t + l16][32 * j + 8 * g]);
        const bf16x8 w1 = get(&Wb[1][16 * t + l16][32 * j + 8 * g]);
        const bf16x8 w2 = get(&Wb[2][16 * t + l16][32 * j + 8 * g]);
        u1 = mfma16(X[j][0], w0, u1);
        u2 = mfma16(X[j][1], w0, u2);
        u1 = mfma16(X[j][0], w1, u1);
        u2 = mfma16(X[j][2], w0, u2);
        u1 = mfma16(X[j][0], w2, u1);
        u2 = mfma16(X[j][1], w1, u2);
      }
      u[t] = (u[t] + (u1 + u2)) * unit;
      const Parts4<3> d = split4<3>(u[t] * out);
#pragma unroll
      for (int z = 0; z < 3; ++z) put(&Vb[z][16 * t + l16][place], d.p[z]);
      const Parts4<3> p = split4<3>(u[t]);
#pragma unroll
      for (int z = 0; z < 3; ++z) put(&Ub[z][16 * t + l16][place], p.p[z]);
    }
    __syncthreads();  // 3
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

// Up to so many rows a request is taken row by row, by a launch of its own where
// others are longer.  us for one request of 32 heads: 6.1, 9.9, 15.1 and 25.5 for 1,
// 4, 8 and 16 rows, 15.5 as a chunk; 16 requests 14, 23, 34 and 57, 73 to 75 as
// chunks; 64 requests 48, 66, 97 and 173, 310 to 316 as chunks.  With few of them
// the second launch (2) costs more than the chunks of short requests, which run
// beside the others.
struct Split {
  int rows;
  bool both;
};
Split split_of(const dft_prompt_gdn_args& a) {
  const bool many = (int64_t)a.batch * a.hv >= 512;
  const int rows = many ? 16 : 7;
  if (a.max_len <= rows) return {rows, false};
  return many && a.cu_seqlens ? Split{rows, true} : Split{0, false};
}
bool all_by_rows(const dft_prompt_gdn_args& a) { return a.max_len <= split_of(a).rows; }
int64_t tiles_of(const dft_prompt_gdn_args& a) { return line_tiles(a.rows, a.batch, kChunk); }

int64_t chunk_blocks(const dft_prompt_gdn_args& a) { return (tiles_of(a) * a.hk + kXcds - 1) / kXcds * kXcds * (a.hv / a.hk); }

int launch_rows(const dft_prompt_gdn_args& a, int most, hipStream_t stream) {
  // With few heads a fourth of the columns each (one request: 5.4 us, 6.5 whole; 64 requests: 57 and 49)
  const int64_t heads = (int64_t)a.batch * a.hv;
  const bool few = heads <= 128, vec = vector_state(a);
  const unsigned blocks = (unsigned)(few ? 4 * heads : heads);
  if (few && vec)
    gdn_rows_kernel<32, true><<<blocks, 256, 0, stream>>>(a, most);
  else if (few)
    gdn_rows_kernel<32, false><<<blocks, 256, 0, stream>>>(a, most);
  else if (vec)
    gdn_rows_kernel<128, true><<<blocks, 256, 0, stream>>>(a, most);
  else
    gdn_rows_kernel<128, false><<<blocks, 256, 0, stream>>>(a, most);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

template <int NT>
int launch_scan(const dft_prompt_gdn_args& a, const Work& work, int past, hipStream_t stream) {
  // by k heads where there is one for every XCD, else by v heads
  const int families = a.batch * (a.batch * a.hk >= kXcds ? a.hk : a.hv);
  const unsigned blocks = (unsigned)((families + kXcds - 1) / kXcds * kXcds * (a.batch * a.hv / families * (8 / NT)));
  const bool bf16 = a.o_dtype == DFT_BF16 && reinterpret_cast<uintptr_t>(a.o) % 8 == 0 && a.o_row_stride % 4 == 0 && a.o_h_stride % 4 == 0;
  if (!vector_state(a))
    gdn_scan_kernel<NT, false, kAnyOut><<<blocks, kScanThreads, 0, stream>>>(a, work, families, past);
  else if (bf16)
    gdn_scan_kernel<NT, true, kBf16Out><<<blocks, kScanThreads, 0, stream>>>(a, work, families, past);
  else
    gdn_scan_kernel<NT, true, kAnyOut><<<blocks, kScanThreads, 0, stream>>>(a, work, families, past);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace

// the most workgroups of a launch, in units of 256 threads
int64_t prompt_gdn_blocks(const dft_prompt_gdn_args* a) {
  // the scan's are three such, and padded to a multiple of the XCDs
  return std::max(((int64_t)a->batch * a->hv + kXcds * a->hv) * 8 * (kScanThreads / 256), all_by_rows(*a) ? 0 : chunk_blocks(*a));
}
int64_t prompt_gdn_workspace(const dft_prompt_gdn_args* a) { return all_by_rows(*a) ? 0 : tiles_of(*a) * a->hv * kHead; }

int launch_prompt_gdn(const dft_prompt_gdn_args* a, hipStream_t stream) {
  const Split split = split_of(*a);
  if (all_by_rows(*a) || split.both) {
    const int st = launch_rows(*a, split.rows, stream);
    if (st != DFT_OK || !split.both) return st;
  }
  const Work work = {static_cast<char*>(a->workspace)};
  gdn_chunk_kernel<<<(unsigned)chunk_blocks(*a), 256, 0, stream>>>(*a, work, split.rows);
  if (hipGetLastError() != hipSuccess) return DFT_ERR_LAUNCH;
  // 16 value columns a workgroup, or 32 at 1.6 times the time a chunk: the longest request's chunks one after the other,
  // or all of them over the CUs (us: one prompt of 8192, 32 heads, 282 and 402; six of 257 to 2999 354 and 302)
  const double longest = std::min(a->rows, (int64_t)a->max_len) / 64.0, all = (a->rows / 64.0 + a->batch / 2.0) * a->hv / kCus;
  return std::max(longest, 8 * all) <= 1.6 * std::max(longest, 4 * all) ? launch_scan<1>(*a, work, split.rows, stream)
                                                                        : launch_scan<2>(*a, work, split.rows, stream);
}

}  // namespace dft
