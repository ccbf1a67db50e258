// Attention of the full-attention layers: dft_paged_attention over a paged
// cache, dft_prompt_attention over whole packed prompts.
//
// A wave per (row, query head): the lanes share head_dim, the keys are taken
// one by one with the running maximum and sum of the softmax.
#include <math.h>
#include <stdint.h>

#include "dft_device.h"

namespace dft {
namespace {

struct Row {
  const void *q, *k, *v;
  int64_t q_off;
};

template <int D, bool PAGED, class Args>
__global__ void __launch_bounds__(64) attend_kernel(Args a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x, h = blockIdx.y, b = blockIdx.z, g = h / (a.hq / a.hkv);
  int span;
  if constexpr (PAGED)
    span = a.n_new;
  else
    span = a.max_len;
  const int64_t r0 = a.cu_seqlens ? a.cu_seqlens[b] : (int64_t)b * span;
  int64_t n = a.cu_seqlens ? (int64_t)a.cu_seqlens[b + 1] - r0 : span;
  int status = n < 0 || n > span || r0 < 0 || r0 + n > a.rows ? DFT_STATUS_SPAN : 0;
  n = min(min(n, (int64_t)span), a.rows - r0);
  if (r0 < 0) n = 0;
  int64_t keys = n;
  if constexpr (PAGED) {
    keys = max(ld_i(a.seq_len, b, a.seq_len_dtype), (int64_t)0);
    if (keys > (int64_t)a.columns * a.page_size) status |= DFT_STATUS_TABLE;
  }
  const int64_t before = keys - n;  // the keys in front of the rows' own (negative: some rows have none)
  if constexpr (PAGED) keys = min(keys, (int64_t)a.columns * a.page_size);
  if (a.status && blockIdx.x == 0 && h == 0 && lane == 0) a.status[b] = status;
  const int64_t i = blockIdx.x;
  if (i >= n) return;
  const int64_t r = r0 + i;

  float q[E], o[E] = {};
  for (int e = 0; e < E; ++e) q[e] = ld_f(a.q, r * a.q_row_stride + h * a.q_h_stride + lane * E + e, a.dtype);
  float top = -INFINITY, sum = 0;
  uint64_t bits = 0;
  if constexpr (PAGED)
    if (a.anc_bits) bits = a.anc_bits[r];
  const int64_t last = a.flags & DFT_ATTN_CAUSAL ? min(before + i + 1, keys) : keys;
  for (int64_t j = 0; j < last; ++j) {
    int64_t ko, vo;
    const void *kp, *vp;
    if constexpr (PAGED) {
      if (a.anc_bits && j >= before && !(bits >> (j - before) & 1)) continue;
      const int page = a.block_table[b * a.table_row_stride + j / a.page_size];
      if (page < 0 || page >= a.num_pages) continue;
      const int64_t t = j % a.page_size;
      ko = page * a.kc_page_stride + t * a.kc_token_stride + g * a.kc_h_stride;
      vo = page * a.vc_page_stride + t * a.vc_token_stride + g * a.vc_h_stride;
      kp = a.key_cache;
      vp = a.value_cache;
    } else {
      ko = (r0 + j) * a.k_row_stride + g * a.k_h_stride;
      vo = (r0 + j) * a.v_row_stride + g * a.v_h_stride;
      kp = a.k;
      vp = a.v;
    }
    float s = 0;
    for (int e = 0; e < E; ++e) s += q[e] * ld_f(kp, ko + lane * E + e, a.dtype);
    for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
    s *= a.scale;
    const float next = fmaxf(top, s);
    const float keep = next == -INFINITY ? 1.f : __expf(top - next), p = next == -INFINITY ? 0.f : __expf(s - next);
    top = next;
    sum = sum * keep + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * keep + p * ld_f(vp, vo + lane * E + e, a.dtype);
  }
  for (int e = 0; e < E; ++e)
    st_f(a.o, r * a.o_row_stride + h * a.o_h_stride + lane * E + e, a.o_dtype, sum > 0 ? o[e] / sum : sum == 0 ? 0 : sum);
  if (a.lse && lane == 0) a.lse[r * a.lse_row_stride + h] = top + logf(sum);
}

template <bool PAGED, class Args>
int launch(const Args& a, int span, hipStream_t stream) {
  const dim3 grid(span, a.hq, a.batch);
  switch (a.head_dim) {
    case 64: attend_kernel<64, PAGED><<<grid, 64, 0, stream>>>(a); break;
    case 128: attend_kernel<128, PAGED><<<grid, 64, 0, stream>>>(a); break;
    default: attend_kernel<256, PAGED><<<grid, 64, 0, stream>>>(a); break;
  }
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace

int64_t paged_attention_workspace(const dft_paged_attention_args* a) { return 0; }
int launch_paged_attention(const dft_paged_attention_args* a, hipStream_t stream) {
  return launch<true>(*a, a->n_new, stream);
}

}  // namespace dft
