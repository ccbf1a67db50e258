// dft_prompt_attention: attention over whole packed prompts.
//
// A workgroup takes 32 NW packed rows (row p: token p / group, head p % group
// of one kv head) of one prompt and walks over the keys they see in tiles of
// 64, which its waves share.  While a tile is worked on the next one is
// copied to the other half of the LDS.
#include "attend.h"

namespace dft {
namespace {

using namespace attend;

template <int D, int NW, class T>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) prompt_kernel(dft_prompt_attention_args a, Scale sc, bool vec) {
  constexpr int kRow = 2 * D, kBytes = kTile * kRow;  // of a tile's keys, and of its values
  constexpr int kRows = 1024 / kRow, kCopies = kTile / (kRows * NW), kPieces = D / 8;
  typedef Rows<D, kTile, T> Wave;
  __shared__ __attribute__((aligned(1024))) char lds[2][2][kBytes];
  __shared__ char notes[NW][Wave::kNotes];
  __shared__ int spoiled;  // the last tile found to hold a value that is not finite
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int group = a.hq / a.hkv;
  const int pairs = a.batch * a.hkv, turn = blockIdx.x / pairs, pair = blockIdx.x - turn * pairs;
  const int b = pair / a.hkv, g = pair - b * a.hkv;

  const int64_t r0 = a.cu_seqlens ? a.cu_seqlens[b] : (int64_t)b * a.max_len;
  int64_t n64 = a.cu_seqlens ? (int64_t)a.cu_seqlens[b + 1] - r0 : a.max_len;
  const bool cut = n64 < 0 || n64 > a.max_len || r0 < 0 || r0 + n64 > a.rows;
  n64 = r0 < 0 ? 0 : min(min(n64, (int64_t)a.max_len), a.rows - r0);
  const int n = (int)max(n64, (int64_t)0);
  if (a.status && turn == 0 && g == 0 && threadIdx.x == 0) a.status[b] = cut ? DFT_STATUS_SPAN : 0;

  // the longest rows first: they see the most keys
  const int p0 = (int)(gridDim.x / pairs - 1 - turn) * 32 * NW, rows = n * group;
  if (p0 >= rows) return;
  const bool causal = a.flags & DFT_ATTN_CAUSAL;
  const int last = (int)((uint32_t)(min(p0 + 32 * NW, rows) - 1) / (uint32_t)group);  // token of the workgroup's last row
  const int keys = causal ? last + 1 : n, tiles = (keys + kTile - 1) / kTile;

  const int pw = p0 + 32 * wave;  // the wave's first row
  const int p = min(pw + (lane & 31), rows - 1);
  const int i = (int)((uint32_t)p / (uint32_t)group), h = g * group + (p - i * group);
  const int limit = causal ? i + 1 : n;  // keys this lane's row sees
  const int least = __builtin_amdgcn_readlane(limit, 0), most = __builtin_amdgcn_readlane(limit, 31);
  const bool works = pw < rows;
  const int fewest = causal ? (int)((uint32_t)p0 / (uint32_t)group) + 1 : n;  // keys that the workgroup's first row sees

  // Copy i of a wave: rows (i NW + wave) kRows ..., the first of them through
  // the scalar base, the lane's through its offset.
  const int lrow = lane / kPieces, piece = lane % kPieces;
  const uint64_t kbase = (uint64_t)(uintptr_t)a.k + 2 * (r0 * a.k_row_stride + g * a.k_h_stride);
  const uint64_t vbase = (uint64_t)(uintptr_t)a.v + 2 * (r0 * a.v_row_stride + g * a.v_h_stride);
  const uint32_t lds0 = lds_address(lds);
  auto copy = [&](int t, int stage) {
    const int j0 = t * kTile;
#pragma unroll
    for (int x = 0; x < kCopies; ++x) {
      const int first = (x * NW + wave) * kRows, row = first + lrow;
      int there = lrow, from = j0 + first;
      if (j0 + kTile > n) {  // the last tile: rows past the prompt become its last row
        from = min(from, n - 1);
        there = min(lrow, n - 1 - from);
      }
      const uint32_t at = lds0 + stage * 2 * kBytes + first * kRow;
      dma16(uniform(kbase + 2 * ((uint64_t)from * a.k_row_stride)),
            (uint32_t)(there * (int)a.k_row_stride * 2 + ((piece ^ key_swizzle<D>(row)) << 4)), at);
      dma16(uniform(vbase + 2 * ((uint64_t)from * a.v_row_stride)),
            (uint32_t)(there * (int)a.v_row_stride * 2 + ((piece ^ value_swizzle<D>(row)) << 4)), at + kBytes);
    }
  };

  Wave w;
  w.clear();
  w.notes = lds_address(notes[wave]);
  if (threadIdx.x == 0) spoiled = -1;
  copy(0, 0);
  w.load_q(static_cast<const uint16_t*>(a.q) + (r0 + i) * a.q_row_stride + h * a.q_h_stride, sc);
  for (int t = 0; t < tiles; ++t) {
    __builtin_amdgcn_s_waitcnt(kWaitDma);
    __syncthreads();
    if (t + 1 < tiles) copy(t + 1, (t + 1) & 1);
    const int j0 = t * kTile;
    const uint32_t at = lds0 + (t & 1) * 2 * kBytes, mine = at + kBytes + wave * (kBytes / NW);
    const bool acts = works && j0 < most, partial = j0 + kTile > least;
    const uint64_t vis = partial ? first_bits(limit - j0) : ~0ull;
    if (j0 + kTile > fewest) {
      if (!finite<T, kBytes / NW>(mine)) spoiled = t;
      __syncthreads();
      if (spoiled == t) {
        if (acts) w.note(at + kBytes, vis);
        __syncthreads();
        clear_infinite<T, kBytes / NW>(mine);
        __syncthreads();
      }
    }
    if (acts) w.tile(at, at + kBytes, sc.c, partial, vis);
  }
  if (!works) return;
  w.finish();
  const float sum = w.whole_sum(), by = weight_of(sum);
  if (pw + (lane & 31) >= rows) return;
  const int64_t to = (r0 + i) * a.o_row_stride + h * a.o_h_stride + 4 * half;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = w.o[t][4 * x + e] * by;
      store4(a.o, to + 32 * t + 8 * x, a.o_dtype, vec, y);
    }
  if (a.lse && half == 0) a.lse[(r0 + i) * a.lse_row_stride + h] = lse_of(w.top, sum);
}

template <int D, class T>
int launch(const dft_prompt_attention_args& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.max_len * (a.hq / a.hkv);
  constexpr int NW = 4;
  const int64_t blocks = (rows + 32 * NW - 1) / (32 * NW) * a.batch * a.hkv;
  if (blocks > 0xffffffffll / (64 * NW)) return DFT_ERR_UNSUPPORTED;  // a grid counts work-items in 32 bits
  prompt_kernel<D, NW, T><<<(unsigned)blocks, 64 * NW, 0, stream>>>(a, split_scale(a.scale), vector_out(a));
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

template <class T>
int launch_type(const dft_prompt_attention_args& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch<64, T>(a, stream);
    case 128: return launch<128, T>(a, stream);
    default: return launch<256, T>(a, stream);
  }
}

}  // namespace

int launch_prompt_attention(const dft_prompt_attention_args* a, hipStream_t stream) {
  return a->dtype == DFT_BF16 ? launch_type<Bf16>(*a, stream) : launch_type<F16>(*a, stream);
}

}  // namespace dft
