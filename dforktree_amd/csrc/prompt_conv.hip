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
constexpr int kRows = 16, kTileRows = 64;  // of a tile, here and in prompt_conv4_kernel

// Workgroups beside each other over the channels (of none: one, for the status).
__host__ __device__ inline int channel_blocks(const dft_prompt_conv_args& p) { return p.channels ? (p.channels + 255) / 256 : 1; }

// The types and strides as they come, a thread a channel: reads and writes of one
// element each, so bound by their number.  The rows of prompt_conv4_kernel's
// figure, with fp32 weights 222 us, all in fp16 267.
__global__ void __launch_bounds__(256) prompt_conv_kernel(const dft_prompt_conv_args p) {
  const int blocks = channel_blocks(p);
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

// Four taps over bf16 rows, outputs and weights, whole pieces of 8 channels a
// thread.  The rows of a tile follow each other through the registers, the next
// four on their way: a row is read once, but for the three in front of each
// tile.  STATE: windows are bf16 as well, [c][3] in one piece.
// The exponential's argument is rounded once, |z| 2^-24 of the value: nothing
// beside the output's 2^-8 (with expf 102 us where it took 82).  Bound by HBM: six
// prompts of 257 to 2999 rows, 8192 channels, 65 us, 4.9 TB/s, 72 over three such
// batches in turn (tiles of 16, 32, 64 and 128 rows 75, 82, 70 and 77; rows read as
// data read once 66).
template <bool STATE>
__global__ void __launch_bounds__(256) prompt_conv4_kernel(const dft_prompt_conv_args p) {
  constexpr int kTile = kTileRows, kAhead = 4;
  typedef __bf16 bf16x8_ __attribute__((ext_vector_type(8)));
  const int blocks = (p.channels / 8 + 255) / 256;
  const int64_t x = blockIdx.x / blocks;
  if (blockIdx.x == 0 && p.status)
    for (int b = threadIdx.x; b < p.batch; b += 256)
      p.status[b] = span_of(p, b).status | slot_of(p.cs_indices, p.cs_indices_dtype, p.initial, p.slots, b).status;
  const int c = ((int)(blockIdx.x - x * blocks) * 256 + threadIdx.x) * 8;
  const bool works = c < p.channels;
  const int cc = works ? c : 0;
  // the weights do not wait for the search
  u32x4 wv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) wv[j] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.weight) + (int64_t)4 * cc + 8 * j);
  const int b = find_tile<256>(p, x, kTile);
  if (b < 0 || !works) return;
  const Span s = span_of(p, b);
  const Slot slot = slot_of(p.cs_indices, p.cs_indices_dtype, p.initial, p.slots, b);
  const int t0 = (int)(x - first_tile(s.r0, b, kTile)) * kTile, t1 = min(t0 + kTile, s.n);
  const uint16_t* rows = static_cast<const uint16_t*>(p.x) + s.r0 * p.x_row_stride + c;
  auto row = [&](int t) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(rows + t * p.x_row_stride)); };

  u32x4 ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) ahead[i] = row(min(t0 + i, t1 - 1));
  // the three inputs in front, as bf16: rows, or the window (element 3 e + j of the thread's 24)
  const int64_t window = slot.at * p.cs_slot_stride + c * p.cs_chan_stride;
  uint16_t in[3][8];
  auto window_at = [&](uint16_t (&w)[24]) {
    if constexpr (STATE) {
      const u32x4* at = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.conv_state) + window);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const u32x4 v = at[i];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[8 * i + e] = (uint16_t)(v[e / 2] >> (e % 2) * 16);
      }
    }
  };
  float f[3][8];
  if (t0 >= 3 || !slot.initial) {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int t = t0 - 3 + j;
      const u32x4 v = t >= 0 ? row(t) : u32x4{};
#pragma unroll
      for (int e = 0; e < 8; ++e) f[j][e] = bf16_bits_to_f32(v[e / 2] >> (e % 2) * 16 & 0xffffu);
    }
  } else {  // t0 is 0
    uint16_t w[24];
    window_at(w);
#pragma unroll
    for (int j = 0; j < 3; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (STATE)
          f[j][e] = bf16_bits_to_f32(w[3 * e + j]);
        else
          f[j][e] = ld_f(p.conv_state, window + e * p.cs_chan_stride + j * p.cs_col_stride, p.cs_dtype);
      }
  }
  if (t0 == 0 && slot.at >= 0) {  // the new window: the last three of the old one and the rows
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int t = s.n - 3 + j;
      const u32x4 v = row(max(t, 0));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float old = t == -2 ? f[1][e] : f[2][e];  // (t is -2 or -1: there is a row)
        const uint16_t now = (uint16_t)(v[e / 2] >> (e % 2) * 16);
        in[j][e] = t >= 0 ? now : bf16_bits(old);
        if constexpr (!STATE) {
          const float left = t >= 0 ? bf16_bits_to_f32(now) : old;
          store(p.conv_state, window + e * p.cs_chan_stride + j * p.cs_col_stride, p.cs_dtype, left);
        }
      }
    }
    if constexpr (STATE) {
      u32x4* at = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.conv_state) + window);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int lo = 8 * i + 2 * e, hi = lo + 1;
          v[e] = (uint32_t)in[lo % 3][lo / 3] | (uint32_t)in[hi % 3][hi / 3] << 16;
        }
        at[i] = v;
      }
    }
  }
  float weight[8][4], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int j = 0; j < 4; ++j) weight[e][j] = bf16_bits_to_f32(wv[e / 2][(e % 2) * 2 + j / 2] >> (j % 2) * 16 & 0xffffu);
    bias[e] = p.bias ? ld_f(p.bias, c + e, p.bias_dtype) : 0.f;
  }
  uint16_t* out = static_cast<uint16_t*>(p.y) + s.r0 * p.y_row_stride + c;
  for (int t = t0; t < t1; t += kAhead) {
    u32x4 now[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) now[i] = ahead[i];
    if (t + kAhead < t1) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ahead[i] = row(min(t + kAhead + i, t1 - 1));
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      bf16x8_ y;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float last = bf16_bits_to_f32(now[i][e / 2] >> (e % 2) * 16 & 0xffffu);
        float acc = fmaf(f[0][e], weight[e][0], bias[e]);
        acc = fmaf(f[1][e], weight[e][1], acc);
        acc = fmaf(f[2][e], weight[e][2], acc);
        acc = fmaf(last, weight[e][3], acc);
        f[0][e] = f[1][e], f[1][e] = f[2][e], f[2][e] = last;
        const float silu = acc * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(acc * -1.4426950408889634f));
        y[e] = (__bf16)(p.silu ? silu : acc);
      }
      if (t + i < t1) *reinterpret_cast<bf16x8_*>(out + (t + i) * p.y_row_stride) = y;
    }
  }
}

bool aligned16(const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; }
// The types and layouts of prompt_conv4_kernel: a layer's own.
bool by_pieces(const dft_prompt_conv_args& a) {
  return a.width == 4 && a.channels && a.channels % 8 == 0 && a.x_dtype == DFT_BF16 && a.y_dtype == DFT_BF16 && a.w_dtype == DFT_BF16 &&
         a.w_tap_stride == 1 && a.w_chan_stride == 4 && aligned16(a.x) && aligned16(a.y) && aligned16(a.weight) &&
         a.x_row_stride % 8 == 0 && a.y_row_stride % 8 == 0;
}
bool window_pieces(const dft_prompt_conv_args& a) {
  return a.cs_dtype == DFT_BF16 && a.cs_col_stride == 1 && a.cs_chan_stride == 3 && a.cs_slot_stride % 8 == 0 && aligned16(a.conv_state);
}

}  // namespace

int64_t prompt_conv_blocks(const dft_prompt_conv_args* a) {
  return line_tiles(a->rows, a->batch, kRows) * channel_blocks(*a);
}

int launch_prompt_conv(const dft_prompt_conv_args* a, hipStream_t stream) {
  if (by_pieces(*a)) {  // fewer workgroups than prompt_conv_blocks
    const unsigned blocks = (unsigned)(line_tiles(a->rows, a->batch, kTileRows) * ((a->channels / 8 + 255) / 256));
    if (window_pieces(*a))
      prompt_conv4_kernel<true><<<blocks, 256, 0, stream>>>(*a);
    else
      prompt_conv4_kernel<false><<<blocks, 256, 0, stream>>>(*a);
    return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
  }
  prompt_conv_kernel<<<(unsigned)prompt_conv_blocks(a), 256, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

}  // namespace dft
