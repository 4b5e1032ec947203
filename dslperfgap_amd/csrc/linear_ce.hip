// Softmax cross entropy of a projection onto a vocabulary, and its gradients, without the
// logits in memory, for gfx950.  With L = logit_scale x W^T (x: tokens x hidden, W: vocab x
// hidden), per token:
//
//   lse = log sum_v exp L_v,  loss = lse - (1 - s) L_label - s / classes sum_v L_v + z lse^2
//   dL_v = dloss logit_scale (exp(L_v - lse) (1 + 2 z lse) - (1 - s) [v = label] - s / classes)
//   dx = dL W,  dW = dL^T x
//
// Forward: the tiles of L stay in the registers that the matrix cores sum them in; a tile
// leaves one (max, sum of exp(L - max)) per token, and the label's logit where it has it.  A
// second kernel joins a token's tiles.  2 tokens hidden vocab operations: bound by the matrix
// cores from a few hundred tokens on, below by the read of W.
//
// Backward, in pieces of the vocabulary: the tiles of L again, dL of the piece rounded to the
// inputs' type into the workspace, then the two products that read it.  (Rounded, because the
// matrix cores take both factors in one type: fp32 ones run at a thirteenth of the 16-bit rate, and
// dL in two 16-bit parts would double both products.)  A piece is as wide as keeps dL within
// kPieceBytes.  dx is summed over pieces, and over parts of a piece where its own tiles are too
// few to fill the card, in fp32 in the workspace, in a fixed order; dW's rows belong to one piece
// each.  No atomics.
//
// Tokens whose label is ignored take no part: the others' rows are numbered first, and where
// any is ignored x is gathered in that order.  What an ignored token's x holds, infinities and
// NaN among it, reaches no output.
//
// dL is scaled by a power of two that brings its largest possible value to 2^14 (taken off again
// where dx and dW are rounded): fp16 then keeps values down to 2^-28 of the largest as normal
// numbers whatever the loss is divided by.  A token of fp16 whose own largest lies below 2^10 then
// has a power of two of its own for dx, whose sums are its alone; ahead of dW, which sums over
// tokens, its dL comes back to the common one.
#include <algorithm>
#include <type_traits>

#include "tile_product.h"
#include "vbh_launch.h"

namespace vbh {

namespace {

constexpr int kRowsLanes = 1024;

// What the kernels behind lce_rows read of it.
struct LceInfo {
  int live;        // tokens that count
  int shift;       // of dL's power of two
  int spread;      // some token's has more of its own (token_shift)
  int splits;      // of a piece's columns in the product that gives dx (dx_splits)
  int split_cols;  // in each
};

// How many workgroups share a tile of dx, each with a part of the piece's columns, so that `tiles`
// tiles of `stages` stages fill the card: by the time of its rounds of workgroups in stages, each
// with kRoundStages for its start and end, and that of the parts' sums, which pass through memory
// in kSumBytes a stage.  At most kSplitRounds rounds of workgroups that share.  One count to a lane
// of a wave.
constexpr int kSplitRounds = 4, kMostSplits = 16, kLeastSplit = 256;
constexpr int kRoundStages = 12, kSumBytes = 4 << 20;
__device__ __forceinline__ int dx_splits(int64_t tiles, int slots, int cols, int value_bytes,
                                         int64_t out_bytes) {
  const int s = (static_cast<int>(threadIdx.x) & (kWave - 1)) + 1;
  if (tiles > kSplitRounds * slots) return 1;
  const int n = static_cast<int>(tiles) * s;
  const int stages = (cols * value_bytes + kStageBytes - 1) / kStageBytes;
  float time = static_cast<float>((n + slots - 1) / slots) *
               static_cast<float>((stages + s - 1) / s + kRoundStages);
  if (s > 1) time += 2.0f * s * static_cast<float>(out_bytes) * (1.0f / kSumBytes);
  if (s > kMostSplits || (s > 1 && (n > kSplitRounds * slots || cols < s * kLeastSplit)))
    time = __builtin_huge_valf();
  float least = time;
  for (int i = 1; i < kWave; i *= 2) least = fminf(least, __shfl_xor(least, i));
  return __builtin_ctzll(__ballot(time == least)) + 1;
}

// |dL| at most of a token with this loss gradient and logsumexp; 0 where that is not finite.
__device__ __forceinline__ float most_dlogit(const LceArgs& a, float dloss, float lse) {
  const float f = 1.0f + 2.0f * a.lse_square_scale * lse;
  const float most = __builtin_fabsf(dloss * a.scale) * (a.target_most + __builtin_fabsf(f));
  return most <= 0x1p127f ? most : 0.0f;
}
// Powers of two that bring a token's dL from the call's scale up to a largest value of 2^kTop: none
// where that is within kNear of it, so that gradients alike in size need no second scale.
constexpr int kTop = 14, kNear = 4;
__device__ __forceinline__ int own_shift(float most, int shift) {
  const int exponent = __builtin_amdgcn_frexp_expf(most) + shift;
  return most > 0.0f && exponent <= kTop - kNear ? kTop - exponent : 0;
}

__device__ __forceinline__ int64_t label_at(const LceArgs& a, int64_t t) {
  const Span s64 = VBH_SPAN(static_cast<const int64_t*>(a.labels), a.tokens);
  const Span s32 = VBH_SPAN(static_cast<const int32_t*>(a.labels), a.tokens);
  if (a.label_i64) {
    const int64_t* p = static_cast<const int64_t*>(a.labels) + t;
    return VBH_IN_SPAN(s64, p, 8) ? *p : 0;
  }
  const int32_t* p = static_cast<const int32_t*>(a.labels) + t;
  return VBH_IN_SPAN(s32, p, 4) ? *p : 0;
}

template <typename T>
__device__ __forceinline__ T load_one(const T* p, const Span& s) {
  return VBH_IN_SPAN(s, p, sizeof(T)) ? *p : T{};
}
template <typename T>
__device__ __forceinline__ void store_one(T* p, T v, const Span& s) {
  if (VBH_IN_SPAN(s, p, sizeof(T))) *p = v;
}

// Numbers the tokens that count: rows[i] is the i-th one's, place[t] token t's number or -1.
// kRowsEach times as many consecutive tokens at a time as the workgroup has lanes, their loads in
// flight together.  Backward: the largest |dL| that a token's dloss, scale and lse allow, and how
// dx's product is shared out.
constexpr int kRowsEach = 8;
constexpr int kRowsWaves = kRowsLanes / kWave;

// Gives the number of tokens that count, to every lane, and, of the kRowsWaves tokens from `line` on,
// their places (`places` in the LDS; -1 where they have none).  The `first` workgroup writes.
__device__ __forceinline__ int number_tokens(const LceArgs& a, bool first, int64_t line, int* places) {
  __shared__ int counts[2][kRowsEach * kRowsWaves];
  __shared__ float most[kRowsWaves], lows[kRowsWaves];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const Span sd = VBH_SPAN(a.dloss, a.tokens), sl = VBH_SPAN(a.lse_in, a.tokens);
  const Span sr = VBH_SPAN(a.rows, a.tokens), sp = VBH_SPAN(a.place, a.tokens);
  const bool sizes = first && a.dloss != nullptr;
  int live = 0, turn = 0;
  float size = 0.0f, least = __builtin_huge_valf();
  for (int64_t chunk = 0; chunk < a.tokens; chunk += kRowsLanes * kRowsEach, turn ^= 1) {
    bool counts_too[kRowsEach];
    float dloss[kRowsEach], lse[kRowsEach];
    const int64_t left = a.tokens - chunk;  // (fewer than a round: its unused parts are skipped)
#pragma unroll
    for (int j = 0; j < kRowsEach; ++j) {
      counts_too[j] = false;
      if (j * kRowsLanes >= left) continue;
      const int64_t t = chunk + j * kRowsLanes + threadIdx.x, at = min(t, a.tokens - 1);
      counts_too[j] = t < a.tokens && label_at(a, at) != a.ignored;
      if (sizes) {
        dloss[j] = load_one(a.dloss + at, sd);
        lse[j] = load_one(a.lse_in + at, sl);
      }
    }
    uint64_t which[kRowsEach];
#pragma unroll
    for (int j = 0; j < kRowsEach; ++j) {
      which[j] = j * kRowsLanes < left ? __ballot(counts_too[j]) : 0;
      if (lane == 0) counts[turn][j * kRowsWaves + wave] = __popcll(which[j]);
      if (!sizes || !counts_too[j]) continue;
      const float b = most_dlogit(a, dloss[j], lse[j]);  // (what is not finite stays as it is)
      size = fmaxf(size, b);
      if (b > 0.0f) least = fminf(least, b);
    }
    __syncthreads();
    // every wave sums up the counts: two of the 128 to a lane
    const int mine = counts[turn][2 * lane], next = counts[turn][2 * lane + 1];
    int sum = mine + next;
    for (int s = 1; s < kWave; s *= 2) {
      const int other = __shfl_up(sum, s);
      if (lane >= s) sum += other;
    }
    const int before = sum - mine - next;
#pragma unroll
    for (int j = 0; j < kRowsEach; ++j) {
      if (j * kRowsLanes >= left) continue;
      const int64_t t = chunk + j * kRowsLanes + threadIdx.x;
      const int slot = j * kRowsWaves + wave;
      const int base = __shfl(before, slot / 2) + (slot & 1 ? __shfl(mine, slot / 2) : 0);
      const int at = live + base + __popcll(which[j] & ((uint64_t(1) << lane) - 1));
      if (t >= a.tokens) continue;
      if (places != nullptr && t >= line && t < line + kRowsWaves)
        places[t - line] = counts_too[j] ? at : -1;
      if (!first) continue;
      store_one(a.place + t, counts_too[j] ? at : -1, sp);
      if (counts_too[j]) store_one(a.rows + at, static_cast<int>(t), sr);
    }
    live += __shfl(sum, kWave - 1);
  }
  for (int s = 1; s < kWave; s *= 2) {
    size = fmaxf(size, __shfl_xor(size, s));
    least = fminf(least, __shfl_xor(least, s));
  }
  if (lane == 0) most[wave] = size, lows[wave] = least;
  __syncthreads();
  if (!first || wave != 0) return live;
  for (int w = 0; w < kRowsWaves; ++w) {
    size = fmaxf(size, most[w]);
    least = fminf(least, lows[w]);
  }
  const int exponent = size > 0.0f ? __builtin_amdgcn_frexp_expf(size) : kTop;
  LceInfo info{live, min(max(kTop - exponent, -120), 100), 0, 1, 0};
  info.spread = a.own_scales && size > 0.0f && own_shift(least, info.shift) > 0;
  if (a.dx != nullptr) {
    const int64_t tiles = static_cast<int64_t>((live + a.dx_rows - 1) / a.dx_rows) * a.dx_cols;
    const int splits = dx_splits(tiles, a.dx_slots, a.first_cols, a.value_bytes,
                                 live * a.padded * 4);
    info.split_cols = (a.first_cols + splits * 128 - 1) / (splits * 128) * 128;
    info.splits = (a.first_cols + info.split_cols - 1) / info.split_cols;
  }
  LceInfo* to = static_cast<LceInfo*>(a.info);
  if (lane == 0) store_one(to, info, VBH_SPAN(to, 1));
  return live;
}

// One workgroup; lce_gather follows.
__global__ __launch_bounds__(kRowsLanes) void lce_rows(const LceArgs a) {
  number_tokens(a, true, 0, nullptr);
}

__device__ __forceinline__ LceInfo lce_info(const LceArgs& a) {
  const LceInfo* info = static_cast<const LceInfo*>(a.info);
  if (info == nullptr) return LceInfo{static_cast<int>(a.tokens), 0, 0, 1, 0};
  return load_one(info, VBH_SPAN(info, 1));
}

// The power of two in token t's dL as dx's product reads it.
template <typename T>
__device__ __forceinline__ int token_shift(const LceArgs& a, const LceInfo& info, int64_t t) {
  if constexpr (std::is_same_v<T, _Float16>) {
    if (info.spread) {
      const float dloss = load_one(a.dloss + t, VBH_SPAN(a.dloss, a.tokens));
      const float lse = load_one(a.lse_in + t, VBH_SPAN(a.lse_in, a.tokens));
      return info.shift + own_shift(most_dlogit(a, dloss, lse), info.shift);
    }
  }
  return info.shift;
}

// x as the products read it: where it lies, or gathered and padded by lce_gather.
template <typename T>
struct LceX {
  const T* p;
  int64_t ld;
  Span span;
  __device__ __forceinline__ LceX(const LceArgs& a, int live) {
    const bool direct = a.x_direct && live == a.tokens;
    p = static_cast<const T*>(direct ? a.x : a.x_packed);
    ld = direct ? a.x_stride : a.padded;
    span = VBH_SPAN(p, (live - 1) * ld + (direct ? a.hidden : a.padded));
  }
};

constexpr int kGatherRows = 4;  // waves of a workgroup, one row each

// One line of `hidden` values to a line of `padded` ones, zeros behind.
template <typename T>
__device__ __forceinline__ void copy_line(const T* from, T* to, int64_t hidden, int64_t padded,
                                          const Span& sf, const Span& st) {
  constexpr int V = Vec<T>::n, kStep = kWave * V, kEach = 4;  // loads in flight
  int64_t c = (threadIdx.x & (kWave - 1)) * V;
  for (; c + (kEach - 1) * kStep + V <= hidden; c += kEach * kStep) {
    typename Raw<T, V>::type raw[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) raw[i] = load_any<T, V, false>(from + c + i * kStep, sf);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      float v[V];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = raw_at<T, V>(raw[i], k);
      store_raw<T, V, false>(to + c + i * kStep, v, st);
    }
  }
  for (; c < padded; c += kStep) {
    float v[V];
    if (c + V <= hidden) {
      const auto raw = load_any<T, V, false>(from + c, sf);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = raw_at<T, V>(raw, k);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] = c + k < hidden ? static_cast<float>(load_one(from + c + k, sf)) : 0.0f;
    }
    store_raw<T, V, false>(to + c, v, st);
  }
}

// Token t's row of x to place `at`; where it has none, zeros for its dx.
template <typename T>
__device__ __forceinline__ void gather_line(const LceArgs& a, int64_t t, int at) {
  if (at >= 0) {
    const T* x = static_cast<const T*>(a.x);
    T* to = static_cast<T*>(a.x_packed);
    copy_line(x + t * a.x_stride, to + at * a.padded, a.hidden, a.padded,
              VBH_SPAN(x, (a.tokens - 1) * a.x_stride + a.hidden),
              VBH_SPAN(to, a.tokens * a.padded));
  } else if (a.dx != nullptr) {
    T* dx = static_cast<T*>(a.dx);
    const Span sd = VBH_SPAN(dx, a.tokens * a.hidden);
    for (int64_t c = threadIdx.x & (kWave - 1); c < a.hidden; c += kWave)
      store_one(dx + t * a.hidden + c, static_cast<T>(0.0f), sd);
  }
}

// x's rows that count, in their order.
template <typename T>
__global__ __launch_bounds__(kGatherRows* kWave) void lce_gather(const LceArgs a) {
  const int live = lce_info(a).live;
  if (live == a.tokens && a.x_direct) return;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kGatherRows + (threadIdx.x >> 6);
  if (t >= a.tokens) return;
  gather_line<T>(a, t, a.place ? load_one(a.place + t, VBH_SPAN(a.place, a.tokens))
                               : static_cast<int>(t));
}

// lce_rows and lce_gather in one, for up to kTogether tokens: every workgroup numbers them all, with
// a row of x to each of its waves (1037 tokens of 2048 fp16 values, forward by 50257 classes over one
// set of inputs: 170 us, with two launches 176; at 8192 tokens the numbering by all of them takes 14 us, by one 7 and the
// other launch 4).
constexpr int kTogether = kRowsLanes * kRowsEach / 2;
template <typename T>
__global__ __launch_bounds__(kRowsLanes) void lce_rows_gather(const LceArgs a) {
  __shared__ int places[kRowsWaves];
  const int64_t line = static_cast<int64_t>(blockIdx.x) * kRowsWaves;
  const int live = number_tokens(a, blockIdx.x == 0, line, places);
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  if ((live == a.tokens && a.x_direct) || line + wave >= a.tokens) return;
  gather_line<T>(a, line + wave, __builtin_amdgcn_readfirstlane(places[wave]));
}

// W's rows at multiples of 16 bytes.
template <typename T>
__global__ __launch_bounds__(kGatherRows* kWave) void lce_pad_weight(const LceArgs a) {
  const int64_t v = static_cast<int64_t>(blockIdx.x) * kGatherRows + (threadIdx.x >> 6);
  if (v >= a.vocab) return;
  const T* w = static_cast<const T*>(a.w_given);
  T* to = static_cast<T*>(a.w_packed);
  copy_line(w + v * a.w_given_stride, to + v * a.padded, a.hidden, a.padded,
            VBH_SPAN(w, (a.vocab - 1) * a.w_given_stride + a.hidden),
            VBH_SPAN(to, a.vocab * a.padded));
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------

// The workgroup's tile of rows x cols tiles.  Consecutive workgroups go to the 8 dies in turn:
// each die takes a run of tiles, kTileRows rows of tiles deep, whose operands its L2 shares.
constexpr int kTileRows = 4;
constexpr int kDies = 8;
struct TileAt {
  int row, col, split;
  bool live;
};
__device__ __forceinline__ TileAt tile_at(int rows, int cols, int splits = 1) {
  const int each_split = rows * cols, n = each_split * splits, each = (n + kDies - 1) / kDies;
  const int i = static_cast<int>(blockIdx.x) / kDies;
  int id = static_cast<int>(blockIdx.x) % kDies * each + i;
  if (i >= each || id >= n) return TileAt{0, 0, 0, false};
  const int split = splits > 1 ? id / each_split : 0;
  id -= split * each_split;
  const int group = id / (kTileRows * cols), in = id - group * kTileRows * cols;
  const int deep = min(kTileRows, rows - group * kTileRows);
  return TileAt{group * kTileRows + in % deep, in / deep, split, true};
}
int64_t tile_grid(int64_t tiles) { return (tiles + kDies - 1) / kDies * kDies; }

struct LsePart {
  float m, s;  // max, sum of exp(L - m): 0 where m is -inf
};
__device__ __forceinline__ float shift_of(float m) { return m == -__builtin_huge_valf() ? 0.0f : m; }
__device__ __forceinline__ LsePart join(const LsePart& a, const LsePart& b) {
  const float m = max_nan(a.m, b.m), by = shift_of(m);
  return LsePart{m, a.s * fast_exp(a.m - by) + b.s * fast_exp(b.m - by)};
}

#define VBH_TILE_BUFFERS(G)                                                     \
  __shared__ __align__(128) char p0[G::kPBuffer], p1[G::kPBuffer], q0[G::kQBuffer], \
      q1[G::kQBuffer]

// Logits of `rows` x `cols` tiles: x's row tiles against W's from `first` on (`cols_left` rows of
// W).  The operands of tile `at`.
template <typename T, typename G>
__device__ __forceinline__ void logits(const LceArgs& a, G& g, const TileAt& at, int live,
                                       int64_t first, int64_t cols_left, char* p0, char* p1,
                                       char* q0, char* q1) {
  const LceX<T> x(a, live);
  const T* w = static_cast<const T*>(a.w);
  const int64_t r0 = static_cast<int64_t>(at.row) * G::BR;
  typename G::P p(x.p + r0 * x.ld, x.ld, live - r0, a.padded, x.span);
  typename G::Q q(w + first * a.w_stride, a.w_stride, cols_left, a.padded,
                  VBH_SPAN(w, (a.vocab - 1) * a.w_stride + a.padded));
  g.run(p, q, a.padded, at.col % G::kFroms, p0, p1, q0, q1);
}

template <typename T, typename G>
__global__ __launch_bounds__(G::kLanes) void lce_forward(const LceArgs a) {
  VBH_TILE_BUFFERS(G);
  const int live = lce_info(a).live;
  const TileAt at = tile_at((live + G::BR - 1) / G::BR, a.col_tiles);
  if (!at.live) return;
  const int64_t c0 = static_cast<int64_t>(at.col) * G::BC;
  G g;
  logits<T>(a, g, at, live, c0, a.vocab - c0, p0, p1, q0, q1);

  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), quarter = lane >> 4;
  const int64_t r0 = static_cast<int64_t>(at.row) * G::BR;
  // columns of the wave's that the vocabulary has (a lane holds those at 4 quarter + i of a block)
  const int left = static_cast<int>(min(a.vocab - c0, static_cast<int64_t>(G::BC))) - g.wave_col();
  LsePart* parts = reinterpret_cast<LsePart*>(p1);           // [WC][BR]
  float* totals = reinterpret_cast<float*>(parts + G::WC * G::BR);  // [WC][BR]
  static_assert(G::WC * G::BR * 12 <= static_cast<int>(sizeof(p1)), "parts fit one buffer");
#pragma unroll
  for (int r = 0; r < G::RB; ++r) {
    const int row = g.wave_row() + r * kBlockRows + (lane & 15);
    // a few blocks at a time: up to 16 logits of a token
    constexpr int kSome = G::CB < 4 ? G::CB : 4;
    LsePart mine{-__builtin_huge_valf(), 0.0f};
    float total = 0.0f;
#pragma unroll
    for (int c = 0; c < G::CB; c += kSome) {
      float v[4 * kSome];
#pragma unroll
      for (int i = 0; i < 4 * kSome; ++i) v[i] = mul_rn(g.sums[r][c + i / 4][i % 4], a.scale);
      if ((c + kSome) * kBlockRows > left) {  // (the vocabulary ends here)
#pragma unroll
        for (int i = 0; i < 4 * kSome; ++i) {
          const bool in = (c + i / 4) * kBlockRows + 4 * quarter + i % 4 < left;
          if (a.smoothing != 0.0f) total += in ? v[i] : 0.0f;
          v[i] = in ? v[i] : -__builtin_huge_valf();
        }
      } else if (a.smoothing != 0.0f) {
#pragma unroll
        for (int i = 0; i < 4 * kSome; ++i) total += v[i];
      }
      float m = mine.m;
#pragma unroll
      for (int i = 0; i < 4 * kSome; ++i) m = max_nan(m, v[i]);
      const float by = shift_of(m);
      float s = mine.s * fast_exp(mine.m - by);
#pragma unroll
      for (int i = 0; i < 4 * kSome; ++i) s += fast_exp(v[i] - by);
      mine = LsePart{m, s};
      __builtin_amdgcn_sched_barrier(0);  // the next ones' values stay out of the registers
    }
    // the label's logit
    const bool own = r0 + row < live;
    const int64_t t = own ? (a.rows ? load_one(a.rows + r0 + row, VBH_SPAN(a.rows, a.tokens))
                                    : static_cast<int>(r0 + row))
                          : 0;
    const int64_t label = own ? label_at(a, t) - a.class_start - c0 - g.wave_col() : -1;
    const bool has = label >= 0 && label < left && label < G::BC / G::WC && ((label >> 2) & 3) == quarter;
    if (__ballot(has) != 0) {
      float v = 0.0f;
#pragma unroll
      for (int c = 0; c < G::CB; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v = label == c * kBlockRows + 4 * quarter + i ? g.sums[r][c][i] : v;
      }
      if (has) store_one(a.picked + r0 + row, v * a.scale, VBH_SPAN(a.picked, a.tokens));
    }
    mine = join(mine, LsePart{swap16_partner(mine.m), swap16_partner(mine.s)});
    mine = join(mine, LsePart{swap32_partner(mine.m), swap32_partner(mine.s)});
    total += swap16_partner(total);
    total += swap32_partner(total);
    if (quarter == 0) {
      const int wc = g.wave_col() / (G::BC / G::WC);
      parts[wc * G::BR + row] = mine;
      totals[wc * G::BR + row] = total;
    }
  }
  __syncthreads();
  const int row = static_cast<int>(threadIdx.x);
  if (row >= G::BR || r0 + row >= live) return;
  LsePart all = parts[row];
  float total = totals[row];
#pragma unroll
  for (int wc = 1; wc < G::WC; ++wc) {
    all = join(all, parts[wc * G::BR + row]);
    total += totals[wc * G::BR + row];
  }
  const int64_t to = at.col * a.tokens + r0 + row;
  LsePart* out = static_cast<LsePart*>(a.parts);
  store_one(out + to, all, VBH_SPAN(out, a.col_tiles * a.tokens));
  if (a.smoothing != 0.0f)
    store_one(a.totals + to, total, VBH_SPAN(a.totals, a.col_tiles * a.tokens));
}

// kJoinRows tokens to a workgroup, each kJoinLanes lanes with every kJoinLanes-th tile: 8 of them in
// a wave, whose parts are joined in it, then 4 waves' through the LDS.
constexpr int kJoinRows = 8;
constexpr int kJoinLanes = 32;

__global__ __launch_bounds__(kJoinRows* kJoinLanes) void lce_join(const LceArgs a) {
  __shared__ LsePart parts[kJoinLanes / 8][kJoinRows];
  __shared__ float totals[kJoinLanes / 8][kJoinRows];
  const int r = static_cast<int>(threadIdx.x) % kJoinRows;
  const int q = static_cast<int>(threadIdx.x) / kJoinRows;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kJoinRows + r;
  const int64_t label = t < a.tokens ? label_at(a, t) : a.ignored;
  const bool counts = t < a.tokens && label != a.ignored;
  const int64_t row = !counts ? 0 : a.place ? load_one(a.place + t, VBH_SPAN(a.place, a.tokens)) : t;
  const LsePart* from = static_cast<const LsePart*>(a.parts);
  const Span sp = VBH_SPAN(from, a.col_tiles * a.tokens);
  const Span st = VBH_SPAN(a.totals, a.col_tiles * a.tokens);
  LsePart all{-__builtin_huge_valf(), 0.0f};
  float total = 0.0f;
  if (counts) {
    for (int64_t k = q; k < a.col_tiles; k += 4 * kJoinLanes) {
      LsePart part[4];  // four tiles' loads in flight
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t at = k + j * kJoinLanes < a.col_tiles ? k + j * kJoinLanes : k;
        part[j] = load_one(from + at * a.tokens + row, sp);
        if (a.smoothing != 0.0f) {
          const float more = load_one(a.totals + at * a.tokens + row, st);
          total += j == 0 || at != k ? more : 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j * kJoinLanes < a.col_tiles) all = join(all, part[j]);
    }
  }
  for (int s = kJoinRows; s < kWave; s *= 2) {
    all = join(all, LsePart{__shfl_xor(all.m, s), __shfl_xor(all.s, s)});
    total += __shfl_xor(total, s);
  }
  if ((threadIdx.x & (kWave - 1)) < kJoinRows) {
    parts[q / 8][r] = all;
    totals[q / 8][r] = total;
  }
  __syncthreads();
  if (q != 0 || t >= a.tokens) return;
  for (int k = 1; k < kJoinLanes / 8; ++k) {
    all = join(all, parts[k][r]);
    total += totals[k][r];
  }
  float loss = 0.0f, lse = 0.0f, z = 0.0f;
  if (counts) {
    // as the sums of exponentials themselves: not a number where every logit is -inf
    lse = all.m == -__builtin_huge_valf() ? __builtin_nanf("") : fast_log(all.s) + all.m;
    const bool hit = label >= a.class_start && label - a.class_start < a.vocab;
    const float base = a.split ? 0.0f : lse;
    const float even = a.smoothing != 0.0f ? total / a.total_classes : 0.0f;
    if (hit)
      loss = base - a.smoothing * even -
             (1.0f - a.smoothing) * load_one(a.picked + row, VBH_SPAN(a.picked, a.tokens));
    else
      loss = a.smoothing != 0.0f ? a.smoothing * (base - even) : 0.0f;
    if (!a.split) {
      z = a.lse_square_scale * lse * lse;
      loss += z;
    }
  }
  store_one(a.loss + t, loss, VBH_SPAN(a.loss, a.tokens));
  store_one(a.lse + t, lse, VBH_SPAN(a.lse, a.tokens));
  store_one(a.z_loss + t, z, VBH_SPAN(a.z_loss, a.tokens));
}

// dL of the piece's columns, scaled, into a.piece: [live][a.pitch], zeros behind the last column.
template <typename T, typename G>
__global__ __launch_bounds__(G::kLanes) void lce_dlogits(const LceArgs a) {
  VBH_TILE_BUFFERS(G);
  const LceInfo info = lce_info(a);
  const TileAt at = tile_at((info.live + G::BR - 1) / G::BR, a.col_tiles);
  if (!at.live) return;
  const int64_t c0 = static_cast<int64_t>(at.col) * G::BC;
  G g;
  logits<T>(a, g, at, info.live, a.first + c0, a.cols - c0, p0, p1, q0, q1);

  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), quarter = lane >> 4;
  const int64_t r0 = static_cast<int64_t>(at.row) * G::BR;
  const int left = static_cast<int>(min(a.cols - c0, static_cast<int64_t>(G::BC))) - g.wave_col();
  const int padded = static_cast<int>(min(a.pitch - c0, static_cast<int64_t>(G::BC))) - g.wave_col();
  const float even = a.smoothing != 0.0f ? a.smoothing / a.total_classes : 0.0f;
  T* piece = static_cast<T*>(a.piece);
  const Span sp = VBH_SPAN(piece, info.live * a.pitch);
#pragma unroll
  for (int r = 0; r < G::RB; ++r) {
    const int row = g.wave_row() + r * kBlockRows + (lane & 15);
    if (r0 + row >= info.live) continue;
    const int64_t t = load_one(a.rows + r0 + row, VBH_SPAN(a.rows, a.tokens));
    const int64_t label = label_at(a, t) - a.class_start - a.first - c0 - g.wave_col();
    const float lse = load_one(a.lse_in + t, VBH_SPAN(a.lse_in, a.tokens));
    const float by = ldexpf(load_one(a.dloss + t, VBH_SPAN(a.dloss, a.tokens)) * a.scale,
                            token_shift<T>(a, info, t));
    const float f = 1.0f + 2.0f * a.lse_square_scale * lse;
    T* to = piece + (r0 + row) * a.pitch + c0 + g.wave_col();
#pragma unroll
    for (int c = 0; c < G::CB; ++c) {
      const int col = c * kBlockRows + 4 * quarter;
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = fast_exp(g.sums[r][c][j] * a.scale - lse);
        float q = fmaf(p, f, -even);
        if (label == col + j) q -= 1.0f - a.smoothing;
        o[j] = col + j < left ? by * q : 0.0f;
      }
      if (col < padded) store_any<T, 4, false>(to + col, o, sp);
    }
  }
}

// Four consecutive values of a line of `n`.
template <typename T>
__device__ __forceinline__ void store_four(T* line, int64_t col, int64_t n, const float (&o)[4],
                                           const Span& s) {
  if (col + 4 <= n) {
    store_any<T, 4, false>(line + col, o, s);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < n) store_any<T, 1, false>(line + col + j, o + j, s);
  }
}

// dW of the piece's rows: dL^T x.
template <typename T, typename G>
__global__ __launch_bounds__(G::kLanes) void lce_dweight(const LceArgs a) {
  VBH_TILE_BUFFERS(G);
  const LceInfo info = lce_info(a);
  const int64_t cols = a.hidden;
  const TileAt at = tile_at(static_cast<int>((a.cols + G::BR - 1) / G::BR),
                            static_cast<int>((cols + G::BC - 1) / G::BC));
  if (!at.live) return;
  const int64_t r0 = static_cast<int64_t>(at.row) * G::BR, c0 = static_cast<int64_t>(at.col) * G::BC;
  const LceX<T> x(a, info.live);
  const T* piece = static_cast<const T*>(a.piece);
  typename G::P p(piece + r0, a.pitch, info.live, a.pitch - r0, VBH_SPAN(piece, info.live * a.pitch));
  typename G::Q q(x.p + c0, x.ld, info.live, a.padded - c0, x.span);
  G g;
  g.run(p, q, info.live, 0, p0, p1, q0, q1);
  T* dw = static_cast<T*>(a.dw);
  const Span sd = VBH_SPAN(dw, a.vocab * a.hidden);
  g.each([&](int row, int col, const f32x4& sums) {
    if (r0 + row >= a.cols) return;
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = ldexpf(sums[j], -info.shift);
    store_four(dw + (a.first + r0 + row) * a.hidden, c0 + col, cols, o, sd);
  });
}

// dx's part from one split's columns of the piece: dL W, into (`more`: onto) the split's fp32 sums,
// [splits][live][padded]; of a single split the last piece's gives dx itself.
template <typename T, typename G>
__global__ __launch_bounds__(G::kLanes) void lce_dx(const LceArgs a, int more, int last) {
  VBH_TILE_BUFFERS(G);
  const LceInfo info = lce_info(a);
  const TileAt at = tile_at((info.live + G::BR - 1) / G::BR,
                            static_cast<int>((a.hidden + G::BC - 1) / G::BC), info.splits);
  if (!at.live) return;
  const int64_t r0 = static_cast<int64_t>(at.row) * G::BR, c0 = static_cast<int64_t>(at.col) * G::BC;
  const int64_t k0 = static_cast<int64_t>(at.split) * info.split_cols;
  const int64_t k = min(a.cols - k0, static_cast<int64_t>(info.split_cols));
  if (k <= 0) return;  // a shorter last piece: those before it have summed into every split
  const T* piece = static_cast<const T*>(a.piece);
  const T* w = static_cast<const T*>(a.w);
  typename G::P p(piece + r0 * a.pitch + k0, a.pitch, info.live - r0,
                  min(a.pitch - k0, static_cast<int64_t>(info.split_cols)),
                  VBH_SPAN(piece, info.live * a.pitch));
  typename G::Q q(w + (a.first + k0) * a.w_stride + c0, a.w_stride, k, a.padded - c0,
                  VBH_SPAN(w, (a.vocab - 1) * a.w_stride + a.padded));
  G g;
  g.run(p, q, k, 0, p0, p1, q0, q1);
  T* dx = static_cast<T*>(a.dx);
  const Span sd = VBH_SPAN(dx, a.tokens * a.hidden);
  const Span ss = VBH_SPAN(a.dx_sums, a.dx_sum_floats);
  const bool direct = last && info.splits == 1;
  g.each([&](int row, int col, const f32x4& sums) {
    if (r0 + row >= info.live || c0 + col >= a.hidden) return;
    float o[4];
    float* to = a.dx_sums +
                (static_cast<int64_t>(at.split) * info.live + r0 + row) * a.padded + c0 + col;
    if (more) {
      load_f32<float, 4>(to, o, ss);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += sums[j];
    if (!direct) {
      store_from_f32<float, 4>(to, o, ss);
      return;
    }
    const int64_t t = load_one(a.rows + r0 + row, VBH_SPAN(a.rows, a.tokens));
    const int shift = token_shift<T>(a, info, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = ldexpf(o[j], -shift);
    store_four(dx + t * a.hidden, c0 + col, a.hidden, o, sd);
  });
}

constexpr int kSumLanes = 256;
constexpr int kSumGroups = 4096;  // at most

// dL of the tokens with powers of two of their own, a row at a time, back to the call's: one more
// rounding where that leaves fp16's normal numbers.  (Backward by 32000 classes, loss gradients alike
// and over 20 powers of two: 2048 tokens of 2048 values 720 and 744 us, 8192 of 4096 5174 and 5290.)
__device__ __forceinline__ void level_piece(const LceArgs& a, const LceInfo& info) {
  typedef _Float16 T;
  constexpr int V = Vec<T>::n;
  T* piece = static_cast<T*>(a.piece);
  const Span sp = VBH_SPAN(piece, info.live * a.pitch);
  for (int64_t row = blockIdx.x; row < info.live; row += gridDim.x) {
    const int64_t t = load_one(a.rows + row, VBH_SPAN(a.rows, a.tokens));
    const int own = token_shift<T>(a, info, t) - info.shift;
    if (own == 0) continue;
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.pitch; c += kSumLanes * V) {
      T* at = piece + row * a.pitch + c;
      const auto raw = load_raw<T, V, false>(at, sp);
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = ldexpf(raw_at<T, V>(raw, k), -own);
      store_raw<T, V, false>(at, o, sp);
    }
  }
}

// dx from the splits' sums behind the last piece, four values of a row to a lane; `level`: the
// piece's dL to the call's scale, for dW.  Launched where nothing is split or levelled too, which only
// the GPU knows (4 us traced).
template <typename T>
__global__ __launch_bounds__(kSumLanes) void lce_dx_join(const LceArgs a, int level, int last) {
  const LceInfo info = lce_info(a);
  if constexpr (std::is_same_v<T, _Float16>) {
    if (level && info.spread) level_piece(a, info);
  }
  if (!last || info.splits == 1) return;
  T* dx = static_cast<T*>(a.dx);
  const Span ss = VBH_SPAN(a.dx_sums, a.dx_sum_floats);
  const int64_t step = info.live * a.padded;
  const uint32_t fours = static_cast<uint32_t>(a.padded / 4);
  for (int64_t row_at = blockIdx.x * int64_t(kSumLanes) + threadIdx.x; row_at < info.live * int64_t(fours);
       row_at += gridDim.x * int64_t(kSumLanes)) {
    // (at most 16 splits of the rows that a few rounds of tiles hold: 32 bits)
    const uint32_t row = static_cast<uint32_t>(row_at) / fours;
    const int64_t c = (static_cast<uint32_t>(row_at) - row * fours) * 4;
    if (c >= a.hidden) continue;
    const int64_t t = load_one(a.rows + row, VBH_SPAN(a.rows, a.tokens));
    const float* from = a.dx_sums + row * a.padded + c;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < info.splits; s += 8) {
      float v[8][4];  // eight splits' loads in flight
#pragma unroll
      for (int i = 0; i < 8; ++i)
        load_f32<float, 4>(from + (s + i < info.splits ? s + i : s) * step, v[i], ss);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += s + i < info.splits ? v[i][j] : 0.0f;
      }
    }
    const int shift = token_shift<T>(a, info, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = ldexpf(o[j], -shift);
    store_four(dx + t * a.hidden, c, a.hidden, o, VBH_SPAN(dx, a.tokens * a.hidden));
  }
}

// dW where there are no tokens at all.
template <typename T>
__global__ __launch_bounds__(kGatherRows* kWave) void lce_zero(T* p, int64_t n) {
  constexpr int kEach = kGatherRows * kWave;
  for (int64_t i = int64_t(blockIdx.x) * kEach + threadIdx.x; i < n; i += int64_t(gridDim.x) * kEach)
    store_one(p + i, static_cast<T>(0.0f), VBH_SPAN(p, n));
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

// Tiles.  A CU's time with a share of n tiles is n times the tile's work over its rate, both against
// kBig's (MI355X, TFLOP/s, bf16 4096 x 8192 x 4096 deep, fp32 2048 x 8192 x 1024):
//   kBig   256 x 256 on 8 waves, one workgroup per CU          1250 (8192 x 8192 x 8192: 1375)
//   kMid   128 x 128 on 4 waves, two per CU                     990, fp32 121
//   kSmall  64 x 128 on 4 waves                                 876, fp32 135
//   kTiny   32 x 128 on 4 waves                                 600, fp32 126
//   kDeep   32 x 64 on 4 waves, three stages ahead: rows by rows of at most 32, whose time is the
//           read of Q
// (The library's best fp32 kernel reaches 118: its matrix instructions take as long as the reads
// for any tile.)
enum Tile { kBig, kMid, kSmall, kTiny, kDeep };
template <typename T, bool P_COLUMNS, bool Q_COLUMNS>
using BigTile = TileProduct<T, 256, 256, 4, 2, P_COLUMNS, Q_COLUMNS>;
template <typename T, bool P_COLUMNS, bool Q_COLUMNS>
using MidTile = TileProduct<T, 128, 128, 2, 2, P_COLUMNS, Q_COLUMNS>;
template <typename T, bool P_COLUMNS, bool Q_COLUMNS>
using SmallTile = TileProduct<T, 64, 128, 2, 2, P_COLUMNS, Q_COLUMNS>;
template <typename T, bool Q_COLUMNS>
using TinyTile = TileProduct<T, 32, 128, 1, 4, false, Q_COLUMNS>;
template <typename T> using DeepTile = TileProduct<T, 32, 64, 2, 2, false, false, true>;

constexpr int64_t kPlainTokens = 64; // a forward of at most these takes one or two rows of tiles
constexpr int64_t kCus = 256;
constexpr int64_t kPieceBytes = int64_t(256) << 20;
constexpr int64_t kPieceCols = 4096; // least of a piece
constexpr int64_t kMostPieceCols = int64_t(1) << 18;

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t tiles(int64_t n, int64_t each) { return (n + each - 1) / each; }
int value_bytes(int dt) { return dt == kF32 ? 4 : 2; }

int64_t tile_rows(Tile t) { return t == kBig ? 256 : t == kMid ? 128 : t == kSmall ? 64 : 32; }
int64_t tile_cols(Tile t) { return t == kBig ? 256 : t == kDeep ? 64 : 128; }
int64_t tile_slots(Tile t) { return t == kBig ? 256 : t == kMid ? 512 : 768; }  // fill the card

// The tile of a product of `rows` by `cols`, whose tiles up to `most_splits` workgroups share;
// P_COLUMNS, Q_COLUMNS: operands with k the slow axis.
Tile tile_of(int64_t rows, int64_t cols, int dt, bool p_columns, bool q_columns,
             int64_t most_splits = 1) {
  if (!p_columns && rows <= 32) return q_columns ? kTiny : kDeep;
  const bool f32 = dt == kF32;
  const struct {
    Tile tile;
    int64_t work;  // percent of kBig's work, over its rate
  } all[] = {{kBig, 100}, {kMid, f32 ? 27 : 31}, {kSmall, f32 ? 13 : 18}, {kTiny, f32 ? 7 : 14}};
  Tile best = kMid;
  int64_t least = int64_t(1) << 62;
  for (const auto& t : all) {
    if (t.tile == kBig ? f32 : p_columns && t.tile > (f32 ? kSmall : kMid)) continue;
    const int64_t n = tiles(rows, tile_rows(t.tile)) * tiles(cols, tile_cols(t.tile));
    const int64_t time = tiles(n * most_splits, kCus) * t.work;
    if (time < least) {
      least = time;
      best = t.tile;
    }
  }
  return best;
}

// Whether a forward numbers the tokens that count: not where dropping the others would leave each
// CU a tile all the same (tokens, hidden, classes in fp32: 300, 768, 5003: 33.8 us, numbered 42.3).
bool numbers(int64_t tokens, int64_t vocab, int dt) {
  const Tile t = tile_of(tokens, vocab, dt, false, false);
  return tokens > kPlainTokens &&
         tiles(tokens, tile_rows(t)) * tiles(vocab, tile_cols(t)) > kCus;
}

// f(TypeTag of the TileProduct)
template <typename T, bool Q_COLUMNS, typename F>
void with_tile(Tile t, F&& f) {
  switch (t) {
    case kBig:
      if constexpr (sizeof(T) == 2) f(TypeTag<BigTile<T, false, Q_COLUMNS>>{});
      break;
    case kMid: f(TypeTag<MidTile<T, false, Q_COLUMNS>>{}); break;
    case kSmall: f(TypeTag<SmallTile<T, false, Q_COLUMNS>>{}); break;
    case kTiny: f(TypeTag<TinyTile<T, Q_COLUMNS>>{}); break;
    case kDeep:
      if constexpr (!Q_COLUMNS) f(TypeTag<DeepTile<T>>{});
      break;
  }
}

// The workspace's parts, each at a multiple of 256 bytes.
struct LcePlan {
  int64_t padded = 0;
  int64_t pieces = 1, piece_cols = 0, pitch = 0;
  int64_t dx_sum_floats = 0;
  Tile dx_tile = kBig;
  int64_t dx_grid = 0;
  int64_t info = 0, rows = 0, place = 0, x = 0, w = 0, parts = 0, totals = 0, picked = 0,
          piece = 0, dx_sums = 0, bytes = 0;
};

LcePlan lce_plan(int64_t tokens, int64_t hidden, int64_t vocab, int dt, bool pad_weight,
                 bool backward) {
  LcePlan p;
  const int64_t e = value_bytes(dt);
  p.padded = up(hidden, 16 / e);
  auto take = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += up(bytes, 256);
    return at;
  };
  p.info = take(sizeof(LceInfo));
  p.rows = take(tokens * 4);
  p.place = take(tokens * 4);
  p.x = take(tokens * p.padded * e);
  if (pad_weight) p.w = take(vocab * p.padded * e);
  if (!backward) {
    const int64_t n = tiles(vocab, tile_cols(tile_of(tokens, vocab, dt, false, false))) * tokens;
    p.parts = take(n * sizeof(LsePart));
    p.totals = take(n * 4);
    p.picked = take(tokens * 4);
    return p;
  }
  // pieces alike in size, of whole tiles
  int64_t most = std::max(kPieceBytes / (tokens * e) / 256 * 256, kPieceCols);
  most = std::min(most, kMostPieceCols);
  p.pieces = tiles(vocab, most);
  p.piece_cols = std::min(up(tiles(vocab, p.pieces), 256), up(vocab, 256));
  p.pieces = tiles(vocab, p.piece_cols);
  p.pitch = up(std::min(p.piece_cols, vocab), 16 / e);
  p.piece = take(tokens * p.pitch * e);
  p.dx_tile = tile_of(tokens, hidden, dt, false, true,
                      std::max<int64_t>(std::min<int64_t>(p.pitch / kLeastSplit, kMostSplits), 1));
  // splits are chosen where the number of tokens that count is known: one, or as many as make
  // kSplitRounds rounds of workgroups at most
  const int64_t br = tile_rows(p.dx_tile), across = tiles(hidden, tile_cols(p.dx_tile));
  const int64_t shared = std::min(kSplitRounds * tile_slots(p.dx_tile) / across * br,
                                  kMostSplits * up(tokens, br));
  p.dx_grid = std::max(tiles(tokens, br) * across, kSplitRounds * tile_slots(p.dx_tile));
  p.dx_sum_floats = std::max(tokens, shared) * p.padded;
  p.dx_sums = take(p.dx_sum_floats * 4);
  return p;
}

unsigned line_groups(const LceArgs& a) {
  return static_cast<unsigned>(tiles(a.tokens, kGatherRows));
}

template <typename T>
hipError_t number_and_gather(const LceArgs& a, hipStream_t s) {
  if (a.tokens <= kTogether) {
    launch_kernel(lce_rows_gather<T>, dim3(static_cast<unsigned>(tiles(a.tokens, kRowsWaves))),
                  dim3(kRowsLanes), 0, s, a);
    return hipGetLastError();
  }
  launch_kernel(lce_rows, dim3(1), dim3(kRowsLanes), 0, s, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  launch_kernel(lce_gather<T>, dim3(line_groups(a)), dim3(kGatherRows * kWave), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t forward(LceArgs a, int dt, bool number, hipStream_t s) {
  hipError_t err = hipSuccess;
  auto done = [&] { return (err = hipGetLastError()) == hipSuccess; };
  if (number) {
    err = number_and_gather<T>(a, s);
  } else if (!a.x_direct) {
    launch_kernel(lce_gather<T>, dim3(line_groups(a)), dim3(kGatherRows * kWave), 0, s, a);
    err = hipGetLastError();
  }
  if (err != hipSuccess) return err;
  const Tile t = tile_of(a.tokens, a.vocab, dt, false, false);
  a.col_tiles = static_cast<int>(tiles(a.vocab, tile_cols(t)));
  with_tile<T, false>(t, [&](auto tag) {
    using G = typename decltype(tag)::type;
    const int64_t grid = tile_grid(tiles(a.tokens, G::BR) * a.col_tiles);
    launch_kernel(lce_forward<T, G>, dim3(static_cast<unsigned>(grid)), dim3(G::kLanes), 0, s, a);
  });
  if (!done()) return err;
  launch_kernel(lce_join, dim3(static_cast<unsigned>(tiles(a.tokens, kJoinRows))),
                dim3(kJoinRows * kJoinLanes), 0, s, a);
  done();
  return err;
}

template <typename T>
hipError_t backward(LceArgs a, int dt, const LcePlan& p, hipStream_t s) {
  hipError_t err = hipSuccess;
  auto done = [&] { return (err = hipGetLastError()) == hipSuccess; };
  if ((err = number_and_gather<T>(a, s)) != hipSuccess) return err;
  for (int64_t i = 0; i < p.pieces; ++i) {
    a.first = i * p.piece_cols;
    a.cols = std::min(p.piece_cols, a.vocab - a.first);
    a.pitch = up(a.cols, 16 / static_cast<int64_t>(sizeof(T)));
    const Tile t = tile_of(a.tokens, a.cols, dt, false, false);
    a.col_tiles = static_cast<int>(tiles(a.cols, tile_cols(t)));
    with_tile<T, false>(t, [&](auto tag) {
      using G = typename decltype(tag)::type;
      const int64_t grid = tile_grid(tiles(a.tokens, G::BR) * a.col_tiles);
      launch_kernel(lce_dlogits<T, G>, dim3(static_cast<unsigned>(grid)), dim3(G::kLanes), 0, s, a);
    });
    if (!done()) return err;
    auto weight = [&] {
      auto go = [&](auto tag) {
        using G = typename decltype(tag)::type;
        const int64_t grid = tile_grid(tiles(a.cols, G::BR) * tiles(a.hidden, G::BC));
        launch_kernel(lce_dweight<T, G>, dim3(static_cast<unsigned>(grid)), dim3(G::kLanes), 0, s,
                      a);
      };
      if constexpr (sizeof(T) == 2) {
        if (tile_of(a.cols, a.hidden, dt, true, true) == kBig) go(TypeTag<BigTile<T, true, true>>{});
        else go(TypeTag<MidTile<T, true, true>>{});
      } else {
        if (tile_of(a.cols, a.hidden, dt, true, true) == kSmall) go(TypeTag<SmallTile<T, true, true>>{});
        else go(TypeTag<MidTile<T, true, true>>{});
      }
      return done();
    };
    const bool last = i + 1 == p.pieces;
    auto rows = [&] {
      with_tile<T, true>(p.dx_tile, [&](auto tag) {
        using G = typename decltype(tag)::type;
        launch_kernel(lce_dx<T, G>, dim3(static_cast<unsigned>(tile_grid(p.dx_grid))),
                      dim3(G::kLanes), 0, s, a, i > 0 ? 1 : 0, last ? 1 : 0);
      });
      return done();
    };
    auto join = [&](bool level) {
      const int64_t groups =
          std::min<int64_t>(tiles(a.tokens * a.padded, 4 * kSumLanes), kSumGroups);
      launch_kernel(lce_dx_join<T>, dim3(static_cast<unsigned>(groups)), dim3(kSumLanes), 0, s, a,
                    level ? 1 : 0, last ? 1 : 0);
      return done();
    };
    if (a.own_scales && a.dw != nullptr) {
      // dx ahead of dW, each with dL at its scale
      if (!rows() || !join(true) || !weight()) return err;
      continue;
    }
    if (a.dw != nullptr && !weight()) return err;
    if (a.dx != nullptr && (!rows() || (last && !join(false)))) return err;
  }
  return err;
}

}  // namespace

int64_t linear_ce_workspace_bytes(int64_t tokens, int64_t hidden, int64_t vocab, int dt,
                                  bool pad_weight, bool backward) {
  // a launch has fewer than 2^32 lanes (the backward's pieces, of 2^36 logits at most, always do)
  const Tile t = tile_of(tokens, vocab, dt, false, false);
  const int64_t lanes = t == kBig ? 512 : 256;
  if (!backward &&
      tile_grid(tiles(tokens, tile_rows(t)) * tiles(vocab, tile_cols(t))) >= (int64_t(1) << 32) / lanes)
    return 0;
  return lce_plan(tokens, hidden, vocab, dt, pad_weight, backward).bytes;
}

hipError_t launch_linear_ce(LceArgs a, int dt, bool back, void* workspace, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (a.tokens == 0) {
    dispatch_float_type(dt, [&](auto tag) {
      using T = typename decltype(tag)::type;
      const int64_t n = a.vocab * a.hidden;
      const int64_t grid = std::min<int64_t>(tiles(n, kGatherRows * kWave), 1 << 16);
      launch_kernel(lce_zero<T>, dim3(static_cast<unsigned>(grid)), dim3(kGatherRows * kWave), 0, s,
                    static_cast<T*>(a.dw), n);
      err = hipGetLastError();
    });
    return err;
  }
  const bool pad_weight = a.w == nullptr;
  const LcePlan p = lce_plan(a.tokens, a.hidden, a.vocab, dt, pad_weight, back);
  char* ws = static_cast<char*>(workspace);
  a.padded = p.padded;
  a.x_packed = ws + p.x;
  const bool number = back || numbers(a.tokens, a.vocab, dt);
  if (number) {
    a.info = ws + p.info;
    a.rows = reinterpret_cast<int*>(ws + p.rows);
    a.place = reinterpret_cast<int*>(ws + p.place);
  }
  if (back) {
    a.piece = ws + p.piece;
    a.dx_sums = reinterpret_cast<float*>(ws + p.dx_sums);
    a.dx_sum_floats = p.dx_sum_floats;
    a.dx_rows = static_cast<int>(tile_rows(p.dx_tile));
    a.dx_cols = static_cast<int>(tiles(a.hidden, tile_cols(p.dx_tile)));
    a.dx_slots = static_cast<int>(tile_slots(p.dx_tile));
    a.first_cols = static_cast<int>(std::min(p.piece_cols, a.vocab));
    a.value_bytes = value_bytes(dt);
    a.own_scales = dt == kF16 && a.dx != nullptr;
  } else {
    a.parts = ws + p.parts;
    a.totals = reinterpret_cast<float*>(ws + p.totals);
    a.picked = reinterpret_cast<float*>(ws + p.picked);
  }
  dispatch_float_type(dt, [&](auto tag) {
    using T = typename decltype(tag)::type;
    if (pad_weight) {
      a.w = a.w_packed = ws + p.w;
      a.w_stride = p.padded;
      launch_kernel(lce_pad_weight<T>, dim3(static_cast<unsigned>(tiles(a.vocab, kGatherRows))),
                    dim3(kGatherRows * kWave), 0, s, a);
      err = hipGetLastError();
      if (err != hipSuccess) return;
    }
    err = back ? backward<T>(a, dt, p, s) : forward<T>(a, dt, number, s);
  });
  return err;
}

}  // namespace vbh
