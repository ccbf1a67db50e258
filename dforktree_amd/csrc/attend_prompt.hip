// dft_prompt_attention: attention over whole packed prompts.
//
// A workgroup takes 32 NW packed rows (row p: token p / group, head p % group
// of one kv head) of one prompt and walks over the keys they see in tiles of
// 64, which its waves share.  A tile's scores are formed beside the tile
// before's weights, so its keys come a tile earlier than its values; the LDS
// holds two tiles of either, one in use, one on its way.  With 128 columns two
// workgroups of four waves share a CU; eight waves on one tile gave 524 us for
// 513.  One prompt of 8192 (32 heads, 8 kv heads, d 128, causal): 515 us, 1.07
// PFLOP/s, the matrix unit busy 63% of the time at the 1.8 GHz that the card's
// power leaves.
#include "attend.h"

namespace dft {
namespace {

using namespace attend;

struct Span {
  int64_t r0;
  int n, status;
};
__device__ __forceinline__ Span span_of(const dft_prompt_attention_args& a, int b) {
  const int64_t r0 = a.cu_seqlens ? a.cu_seqlens[b] : (int64_t)b * a.max_len;
  int64_t n = a.cu_seqlens ? (int64_t)a.cu_seqlens[b + 1] - r0 : a.max_len;
  const bool cut = n < 0 || n > a.max_len || r0 < 0 || r0 + n > a.rows;
  n = r0 < 0 ? 0 : min(min(n, (int64_t)a.max_len), a.rows - r0);
  return {r0, (int)max(n, (int64_t)0), cut ? DFT_STATUS_SPAN : 0};
}

// Row tile `tile` of request b and kv head g.
struct Item {
  int b, g, tile;
  Span span;
};

// Packed prompts of different lengths: the workgroup's item where those of
// all requests stand by falling row tile, so that the first workgroups get
// the most keys and none of them the tiles that a shorter prompt has not got
// (six prompts of 257 to 2999 tokens, by request instead, nearly half of them
// of that kind and spread over the grid: 228 us, so 197).  False past
// the last one.  Each wave finds it for itself: a lane holds a request and
// tries a tile, 64 at a time.  From 65 requests on that would cost more than
// it gives.
constexpr int kSorted = 64;
template <int BM>
__device__ __forceinline__ bool sorted_item(const dft_prompt_attention_args& a, int group, int most, Item& item) {
  const int lane = threadIdx.x & 63;
  Span span = span_of(a, min(lane, a.batch - 1));
  if (a.status && blockIdx.x == 0 && threadIdx.x < a.batch) a.status[threadIdx.x] = span.status;
  const uint32_t tiles = lane < a.batch ? (uint32_t)(span.n * group + BM - 1) / BM : 0;
  auto from = [&](uint32_t tile) {  // items of row tile `tile` or later, of one kv head
    uint32_t sum = 0;
    for (int i = 0; i < a.batch; ++i) sum += __builtin_elementwise_sub_sat((uint32_t)__builtin_amdgcn_readlane(tiles, i), tile);
    return sum;
  };
  uint32_t x = blockIdx.x / a.hkv, low = 0;
  item.g = blockIdx.x - x * a.hkv;
  const uint32_t first = __builtin_amdgcn_readlane(tiles, 0);
  if (__ballot(lane < a.batch && tiles != first) == 0) {  // all alike
    const uint32_t turn = x / a.batch;
    if (turn >= first) return false;
    item.b = x - turn * a.batch;
    low = first - 1 - turn;
  } else {
    for (uint32_t width = most, step = 0; step != 1; width = step) {  // the last tile that more than x items come from
      step = (width + 63) / 64;
      const uint64_t more = __ballot(from(low + lane * step) > x);
      if (!more) return false;
      low += (__popcll(more) - 1) * step;
    }
    uint64_t has = __ballot(tiles > low);
    for (x -= __builtin_amdgcn_readfirstlane(from(low + 1)); x; --x) has &= has - 1;
    item.b = __ffsll((unsigned long long)has) - 1;
  }
  item.tile = (int)low;
  item.span.n = __builtin_amdgcn_readlane(span.n, item.b);
  item.span.r0 = __builtin_amdgcn_readlane((int)span.r0, item.b);
  return true;
}

template <int D, int NW, class T>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) prompt_kernel(dft_prompt_attention_args a, Scale sc, bool vec) {
  constexpr int kRow = 2 * D, kBytes = kTile * kRow;  // of a tile's keys, and of its values
  constexpr int kRows = 1024 / kRow, kCopies = kTile / (kRows * NW), kPieces = D / 8;
  typedef Rows<D, kTile, T> Wave;
  __shared__ __attribute__((aligned(1024))) char keys_at[2][kBytes], values_at[2][kBytes];
  __shared__ char notes[NW][Wave::kNotes];
  __shared__ int spoiled;  // the last tile found to hold a value that is not finite
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int group = a.hq / a.hkv;
  const int pairs = a.batch * a.hkv;
  Item item;
  if (a.cu_seqlens && a.batch > 1 && a.batch <= kSorted) {
    if (!sorted_item<32 * NW>(a, group, gridDim.x / pairs, item)) return;
  } else {
    // the longest rows first: they see the most keys
    const int turn = blockIdx.x / pairs, pair = blockIdx.x - turn * pairs;
    item.b = pair / a.hkv;
    item.g = pair - item.b * a.hkv;
    item.tile = (int)(gridDim.x / pairs) - 1 - turn;
    item.span = span_of(a, item.b);
    if (a.status && turn == 0 && item.g == 0 && threadIdx.x == 0) a.status[item.b] = item.span.status;
  }
  const int g = item.g;
  const int64_t r0 = item.span.r0;
  const int n = item.span.n, p0 = item.tile * 32 * NW, rows = n * group;
  if (p0 >= rows) return;
  const bool causal = a.flags & DFT_ATTN_CAUSAL;
  const int last = (int)((uint32_t)(min(p0 + 32 * NW, rows) - 1) / (uint32_t)group);  // token of the workgroup's last row
  const int keys = causal ? last + 1 : n, tiles = (keys + kTile - 1) / kTile;

  const int pw = p0 + 32 * wave;  // the wave's first row
  const int p = min(pw + (lane & 31), rows - 1);
  const int i = (int)((uint32_t)p / (uint32_t)group), h = g * group + (p - i * group);
  const int limit = causal ? i + 1 : n;  // keys this lane's row sees
  const int least = __builtin_amdgcn_readlane(limit, 0);
  const bool works = pw < rows;
  const int fewest = causal ? (int)((uint32_t)p0 / (uint32_t)group) + 1 : n;  // keys that the workgroup's first row sees

  // Copy x of a wave: the kRows rows of the tile from (x NW + wave) kRows on,
  // the first of them through the scalar base, the lane's through its offset.
  const int piece = lane % kPieces;
  const uint64_t kbase = (uint64_t)(uintptr_t)a.k + 2 * (r0 * a.k_row_stride + g * a.k_h_stride);
  const uint64_t vbase = (uint64_t)(uintptr_t)a.v + 2 * (r0 * a.v_row_stride + g * a.v_h_stride);
  auto ktile = [&](int t) { return lds_address(keys_at) + (t & 1) * kBytes; };
  auto vtile = [&](int t) { return lds_address(values_at) + (t & 1) * kBytes; };
  uint32_t koff[kCopies], voff[kCopies];
  auto offsets = [&](int last) {  // rows past `last` become it
#pragma unroll
    for (int x = 0; x < kCopies; ++x) {
      const int row = (x * NW + wave) * kRows + lane / kPieces, there = min(row, last);
      koff[x] = (uint32_t)(there * (int)a.k_row_stride * 2 + ((piece ^ key_swizzle<D>(row)) << 4));
      voff[x] = (uint32_t)(there * (int)a.v_row_stride * 2 + ((piece ^ value_swizzle<D>(row)) << 4));
    }
  };
  // keys of tile t, or values; the last tile's rows end with the prompt
  auto copy_keys = [&](int t) {
    if ((t + 1) * kTile > n) offsets(n - 1 - t * kTile);
    dma16<kCopies, 1024 * NW>(kbase + (uint64_t)t * (2 * kTile * a.k_row_stride), koff, ktile(t) + 1024 * wave);
  };
  auto copy_values = [&](int t) {
    dma16<kCopies, 1024 * NW>(vbase + (uint64_t)t * (2 * kTile * a.v_row_stride), voff, vtile(t) + 1024 * wave);
  };

  Wave w;
  w.clear();
  w.notes = lds_address(notes[wave]);
  if (threadIdx.x == 0) spoiled = -1;
  offsets(kTile - 1);
  copy_keys(0);
  copy_values(0);
  if (tiles > 1) copy_keys(1);
  w.load_q(static_cast<const uint16_t*>(a.q) + (r0 + i) * a.q_row_stride + h * a.q_h_stride, sc);
  __builtin_amdgcn_s_waitcnt(kWaitDma);
  __syncthreads();
  // of tile t: the keys that the lane's row sees, whether some row of the wave misses some
  auto seen = [&](int t) { return first_bits(limit - t * kTile); };
  auto partial = [&](int t) { return (t + 1) * kTile > least; };
  // what of its values is not finite must not reach a row that does not see it
  auto look = [&](int t) {
    if ((t + 1) * kTile <= fewest) return;
    const uint32_t v = vtile(t), mine = v + wave * (kBytes / NW);
    if (!finite<T, kBytes / NW>(mine)) spoiled = t;
    __syncthreads();
    if (spoiled == t) {
      w.note(v, seen(t));
      __syncthreads();
      clear_infinite<T, kBytes / NW>(mine);
      __syncthreads();
    }
  };
  typename Wave::Scores s;
  w.scores(ktile(0), s);
  if (partial(0)) w.mask(s, seen(0));
  __syncthreads();  // tile 2's keys take the place of tile 0's
  for (int t = 0; t + 1 < tiles; ++t) {
    copy_values(t + 1);
    if (t + 2 < tiles) copy_keys(t + 2);
    look(t);
    w.template step<true>(ktile(t + 1), vtile(t), sc.c, s, [](int) {});
    if (partial(t + 1)) w.mask(s, seen(t + 1));
    __builtin_amdgcn_s_waitcnt(kWaitDma);
    __syncthreads();
  }
  look(tiles - 1);
  w.template step<false>(0, vtile(tiles - 1), sc.c, s, [](int) {});
  if (!works) return;
  w.finish();
  const float sum = w.whole_sum(), by = weight_of(sum);
  if (pw + (lane & 31) >= rows) return;
  w.store(a.o, (r0 + i) * a.o_row_stride + h * a.o_h_stride, a.o_dtype, vec, by);
  if (a.lse && half == 0) a.lse[(r0 + i) * a.lse_row_stride + h] = lse_of(w.top, sum);
}

// The status words of a launch without rows.
__global__ void __launch_bounds__(256) status_kernel(dft_prompt_attention_args a) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.batch) a.status[b] = span_of(a, b).status;
}

// A grid has the row tiles of the longest prompt for every prompt and counts
// work-items in 32 bits: packed batches that need more go in several launches.
template <int D, class T>
int launch(const dft_prompt_attention_args& args, hipStream_t stream) {
  constexpr int NW = 4;
  constexpr int64_t kMost = 0xffffffffll / (64 * NW);
  dft_prompt_attention_args a = args;
  if (a.cu_seqlens && a.max_len > a.rows) a.max_len = (int)a.rows;  // longer ones end past the rows and are cut to them
  const int64_t rows = (int64_t)a.max_len * (a.hq / a.hkv);
  const int64_t each = (rows + 32 * NW - 1) / (32 * NW) * a.hkv;
  int64_t per = a.batch;
  if (per * each > kMost) {
    per = kMost / each;
    if (!per || !a.cu_seqlens) return DFT_ERR_UNSUPPORTED;
  }
  const Scale scale = split_scale(a.scale);
  for (int64_t b = 0; b < args.batch; b += per) {
    a.batch = (int)(args.batch - b < per ? args.batch - b : per);
    prompt_kernel<D, NW, T><<<(unsigned)(each * a.batch), 64 * NW, 0, stream>>>(a, scale, vector_out(a));
    if (hipGetLastError() != hipSuccess) return DFT_ERR_LAUNCH;
    if (a.cu_seqlens) a.cu_seqlens += a.batch;
    if (a.status) a.status += a.batch;
  }
  return DFT_OK;
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

int launch_prompt_status(const dft_prompt_attention_args* a, hipStream_t stream) {
  status_kernel<<<(a->batch + 255) / 256, 256, 0, stream>>>(*a);
  return hipGetLastError() == hipSuccess ? DFT_OK : DFT_ERR_LAUNCH;
}

int launch_prompt_attention(const dft_prompt_attention_args* a, hipStream_t stream) {
  return a->dtype == DFT_BF16 ? launch_type<Bf16>(*a, stream) : launch_type<F16>(*a, stream);
}

}  // namespace dft
