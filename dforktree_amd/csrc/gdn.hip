// dft_prompt_gdn: the gated delta rule over packed prompts and single tokens.
//
// Per v head and row, q and k normalised, q scaled:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q
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

// Whether a state's columns are read in 16-byte pieces.
bool vector_state(const dft_prompt_gdn_args& a) {
  return a.state_k_stride == 1 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0 && a.state_v_stride % 4 == 0 &&
         a.state_h_stride % 4 == 0 && a.state_slot_stride % 4 == 0;
}

}  // namespace

int64_t prompt_gdn_blocks(const dft_prompt_gdn_args* a) { return (int64_t)a->batch * a->hv * 4; }
int64_t prompt_gdn_workspace(const dft_prompt_gdn_args* a) { return 0; }

int launch_prompt_gdn(const dft_prompt_gdn_args* a, hipStream_t stream) {
  const unsigned blocks = (unsigned)(a->batch * a->hv);
  if (vector_state(*a))
    gdn_rows_kernel<128, true><<<blocks, 256, 0, stream>>>(*a);
  else
    gdn_rows_kernel<128, false><<<blocks, 256, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace dft
