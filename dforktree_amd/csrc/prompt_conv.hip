// dft_prompt_conv: the causal convolution in front of a GDN layer, over packed
// prompts or single tokens, with the requests' windows.
//
//   y_t[c] = act(sum_j w[c][j] x_{t-W+1+j}[c] + bias[c])
//
// HBM-bound: an element is read and written once, 2 W operations between.  A
// workgroup takes a tile of rows of one request and a block of channels; the W
// - 1 rows in front of the tile are its own request's, or its window.  The
// workgroup of a request's first tile alone reads the window, and writes the
// new one once it has read the old: no other one touches it.
#include "packed.h"

namespace dft {
namespace {

using namespace packed;

constexpr int kMaxTaps = 8;
constexpr int kRows = 16;  // of a tile

// The types and strides as they come, a thread a channel.
__global__ void __launch_bounds__(256) prompt_conv_kernel(const dft_prompt_conv_args p) {
  const int blocks = (p.channels + 255) / 256;
  const int64_t x = blockIdx.x / blocks;
  if (blockIdx.x == 0 && p.status)
    for (int b = threadIdx.x; b < p.batch; b += 256)
      p.status[b] = span_of(p, b).status | slot_of(p.cs_indices, p.cs_indices_dtype, p.initial, p.slots, b).status;
  const int b = find_tile<256>(p, x, kRows);
  if (b < 0) return;
  const int c = (int)(blockIdx.x - x * blocks) * 256 + threadIdx.x;
  if (c >= p.channels) return;
  const Span s = span_of(p, b);
  const Slot slot = slot_of(p.cs_indices, p.cs_indices_dtype, p.initial, p.slots, b);
  const int W = p.width, t0 = (int)(x - first_tile(s.r0, b, kRows)) * kRows, t1 = min(t0 + kRows, s.n);

  const int64_t window = slot.at * p.cs_slot_stride + c * p.cs_chan_stride;
  auto input = [&](int t) {  // the request's input t, from its window for t < 0
    if (t >= 0) return ld_f(p.x, (s.r0 + t) * p.x_row_stride + c, p.x_dtype);
    return slot.initial ? ld_f(p.conv_state, window + (t + W - 1) * p.cs_col_stride, p.cs_dtype) : 0.f;
  };
  float w[kMaxTaps], in[kMaxTaps];
#pragma unroll
  for (int j = 0; j < kMaxTaps; ++j) {
    w[j] = j < W ? ld_f(p.weight, c * p.w_chan_stride + j * p.w_tap_stride, p.w_dtype) : 0.f;
    in[j] = j < W - 1 ? input(t0 - (W - 1) + j) : 0.f;
  }
  const float bias = p.bias ? ld_f(p.bias, c, p.bias_dtype) : 0.f;
  for (int t = t0; t < t1; ++t) {
    const float now = input(t);
    float acc = bias;
#pragma unroll
    for (int j = 0; j < kMaxTaps; ++j) {
      if (j == W - 1) in[j] = now;
      if (j < W) acc = fmaf(in[j], w[j], acc);
    }
    store(p.y, (s.r0 + t) * p.y_row_stride + c, p.y_dtype, p.silu ? acc / (1.f + expf(-acc)) : acc);
#pragma unroll
    for (int j = 0; j + 1 < kMaxTaps; ++j) in[j] = in[j + 1];
  }
  if (t0 == 0 && slot.at >= 0) {
    float left[kMaxTaps];
#pragma unroll
    for (int j = 0; j < kMaxTaps - 1; ++j) left[j] = j < W - 1 ? input(s.n - (W - 1) + j) : 0.f;
#pragma unroll
    for (int j = 0; j < kMaxTaps - 1; ++j)
      if (j < W - 1) store(p.conv_state, window + j * p.cs_col_stride, p.cs_dtype, left[j]);
  }
}

}  // namespace

int64_t prompt_conv_blocks(const dft_prompt_conv_args* a) {
  return line_tiles(a->rows, a->batch, kRows) * ((a->channels + 255) / 256);
}

int launch_prompt_conv(const dft_prompt_conv_args* a, hipStream_t stream) {
  prompt_conv_kernel<<<(unsigned)prompt_conv_blocks(a), 256, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace dft
