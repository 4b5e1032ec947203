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
// inputs' type into the workspace, then the two products that read it.  A piece is as wide as
// keeps dL within kPieceBytes.  dx is summed over pieces, and over parts of a piece where its
// own tiles are too few to fill the card, in fp32 in the workspace, in a fixed order; dW's rows
// belong to one piece each.  No atomics.
//
// Tokens whose label is ignored take no part: the others' rows are numbered first, and where
// any is ignored x is gathered in that order.  What an ignored token's x holds, infinities and
// NaN among it, reaches no output.
//
// dL is scaled by a power of two that brings its largest possible value to 2^10 (taken off again
// where dx and dW are rounded): fp16 then keeps probabilities down to 2^-24 of the largest as
// normal numbers whatever the loss is divided by.
#include <algorithm>

#include "tile_product.h"
#include "vbh_launch.h"

namespace vbh {

namespace {

constexpr int kRowsLanes = 1024;

// What the kernels behind lce_rows read of it.
struct LceInfo {
  int live;    // tokens that count
  int shift;   // of dL's power of two
};

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
// One workgroup, each lane a run of consecutive tokens.  Backward: the largest |dL| that a
// token's dloss, scale and lse allow.
__global__ __launch_bounds__(kRowsLanes) void lce_rows(const LceArgs a) {
  __shared__ int counts[kRowsLanes / kWave];
  __shared__ float most[kRowsLanes / kWave];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int64_t each = (a.tokens + kRowsLanes - 1) / kRowsLanes;
  const int64_t first = min(each * threadIdx.x, a.tokens), last = min(first + each, a.tokens);
  const Span sd = VBH_SPAN(a.dloss, a.tokens), sl = VBH_SPAN(a.lse_in, a.tokens);
  const Span sr = VBH_SPAN(a.rows, a.tokens), sp = VBH_SPAN(a.place, a.tokens);
  int count = 0;
  float size = 0.0f;
  for (int64_t t = first; t < last; ++t) {
    if (label_at(a, t) == a.ignored) continue;
    ++count;
    if (a.dloss == nullptr) continue;
    const float f = 1.0f + 2.0f * a.lse_square_scale * load_one(a.lse_in + t, sl);
    const float b = __builtin_fabsf(load_one(a.dloss + t, sd) * a.scale) * (1.0f + __builtin_fabsf(f));
    if (b <= 0x1p127f) size = fmaxf(size, b);  // what is not finite stays as it is
  }
  int before = count;
  for (int s = 1; s < kWave; s *= 2) {
    const int other = __shfl_up(before, s);
    if (lane >= s) before += other;
    size = fmaxf(size, __shfl_xor(size, s));
  }
  if (lane == kWave - 1) {
    counts[wave] = before;
    most[wave] = size;
  }
  before -= count;
  __syncthreads();
  int live = 0;
  size = 0.0f;
  for (int w = 0; w < kRowsLanes / kWave; ++w) {
    if (w < wave) before += counts[w];
    live += counts[w];
    size = fmaxf(size, most[w]);
  }
  for (int64_t t = first; t < last; ++t) {
    const bool counts_too = label_at(a, t) != a.ignored;
    store_one(a.place + t, counts_too ? before : -1, sp);
    if (counts_too) store_one(a.rows + before++, static_cast<int>(t), sr);
  }
  if (threadIdx.x == 0) {
    LceInfo* info = static_cast<LceInfo*>(a.info);
    const Span si = VBH_SPAN(info, 1);
    const int exponent = size > 0.0f ? __builtin_amdgcn_frexp_expf(size) : 10;
    store_one(info, LceInfo{live, min(max(10 - exponent, -100), 100)}, si);
  }
}

__device__ __forceinline__ LceInfo lce_info(const LceArgs& a) {
  const LceInfo* info = static_cast<const LceInfo*>(a.info);
  if (info == nullptr) return LceInfo{static_cast<int>(a.tokens), 0};
  return load_one(info, VBH_SPAN(info, 1));
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
  constexpr int V = Vec<T>::n;
  for (int64_t c = (threadIdx.x & (kWave - 1)) * V; c < padded; c += kWave * V) {
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

// x's rows that count, in their order, and zeros for dx of the others.
template <typename T>
__global__ __launch_bounds__(kGatherRows* kWave) void lce_gather(const LceArgs a) {
  const int live = lce_info(a).live;
  if (live == a.tokens && a.x_direct) return;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kGatherRows + (threadIdx.x >> 6);
  if (t >= a.tokens) return;
  const int at = a.place ? load_one(a.place + t, VBH_SPAN(a.place, a.tokens)) : static_cast<int>(t);
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
  int row, col;
  bool live;
};
__device__ __forceinline__ TileAt tile_at(int rows, int cols) {
  const int n = rows * cols, each = (n + kDies - 1) / kDies;
  const int i = static_cast<int>(blockIdx.x) / kDies;
  const int id = static_cast<int>(blockIdx.x) % kDies * each + i;
  if (i >= each || id >= n) return TileAt{0, 0, false};
  const int group = id / (kTileRows * cols), in = id - group * kTileRows * cols;
  const int deep = min(kTileRows, rows - group * kTileRows);
  return TileAt{group * kTileRows + in % deep, in / deep, true};
}
int64_t tile_grid(int64_t rows, int64_t cols) { return (rows * cols + kDies - 1) / kDies * kDies; }

struct LsePart {
  float m, s;  // max, sum of exp(L - m): 0 where m is -inf
};
__device__ __forceinline__ float shift_of(float m) { return m == -__builtin_huge_valf() ? 0.0f : m; }
__device__ __forceinline__ LsePart join(const LsePart& a, const LsePart& b) {
  const float m = max_nan(a.m, b.m), by = shift_of(m);
  return LsePart{m, a.s * fast_exp(a.m - by) + b.s * fast_exp(b.m - by)};
}

#define VBH_TILE_BUFFERS(G)                                                         \
  __shared__ __align__(128) char p0[G::P::kBytes], p1[G::P::kBytes], q0[G::Q::kBytes], \
      q1[G::Q::kBytes]

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
  g.run(p, q, a.padded, p0, p1, q0, q1);
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

// One token per group of kJoinLanes lanes of a workgroup, each with every kJoinLanes-th tile.
constexpr int kJoinRows = 32;
constexpr int kJoinLanes = 32;

__global__ __launch_bounds__(kJoinRows* kJoinLanes) void lce_join(const LceArgs a) {
  __shared__ LsePart parts[kJoinLanes][kJoinRows];
  __shared__ float totals[kJoinLanes][kJoinRows];
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
    for (int64_t k = q; k < a.col_tiles; k += kJoinLanes) {
      all = join(all, load_one(from + k * a.tokens + row, sp));
      if (a.smoothing != 0.0f) total += load_one(a.totals + k * a.tokens + row, st);
    }
  }
  parts[q][r] = all;
  totals[q][r] = total;
  __syncthreads();
  if (q != 0 || t >= a.tokens) return;
  for (int k = 1; k < kJoinLanes; ++k) {
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
    const float by = ldexpf(load_one(a.dloss + t, VBH_SPAN(a.dloss, a.tokens)) * a.scale, info.shift);
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
  g.run(p, q, info.live, p0, p1, q0, q1);
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

// dx's part from the piece's columns of split blockIdx.y: dL W.  One split and one piece: dx
// itself; else into (`more`: onto) the split's fp32 sums.
template <typename T, typename G>
__global__ __launch_bounds__(G::kLanes) void lce_dx(const LceArgs a, int more) {
  VBH_TILE_BUFFERS(G);
  const LceInfo info = lce_info(a);
  const TileAt at = tile_at((info.live + G::BR - 1) / G::BR,
                            static_cast<int>((a.hidden + G::BC - 1) / G::BC));
  if (!at.live) return;
  const int64_t r0 = static_cast<int64_t>(at.row) * G::BR, c0 = static_cast<int64_t>(at.col) * G::BC;
  const int64_t k0 = blockIdx.y * a.split_cols, k = min(a.cols - k0, a.split_cols);
  const T* piece = static_cast<const T*>(a.piece);
  const T* w = static_cast<const T*>(a.w);
  typename G::P p(piece + r0 * a.pitch + k0, a.pitch, info.live - r0,
                  min(a.pitch - k0, a.split_cols), VBH_SPAN(piece, info.live * a.pitch));
  typename G::Q q(w + (a.first + k0) * a.w_stride + c0, a.w_stride, k, a.padded - c0,
                  VBH_SPAN(w, (a.vocab - 1) * a.w_stride + a.padded));
  G g;
  g.run(p, q, k, p0, p1, q0, q1);
  T* dx = static_cast<T*>(a.dx);
  const Span sd = VBH_SPAN(dx, a.tokens * a.hidden);
  const Span ss = VBH_SPAN(a.dx_sums, a.splits * a.tokens * a.padded);
  g.each([&](int row, int col, const f32x4& sums) {
    if (r0 + row >= info.live || c0 + col >= a.hidden) return;
    float o[4];
    if (a.dx_sums == nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = ldexpf(sums[j], -info.shift);
      const int64_t t = load_one(a.rows + r0 + row, VBH_SPAN(a.rows, a.tokens));
      store_four(dx + t * a.hidden, c0 + col, a.hidden, o, sd);
      return;
    }
    float* to = a.dx_sums + (blockIdx.y * a.tokens + r0 + row) * a.padded + c0 + col;
    if (more) {
      load_f32<float, 4>(to, o, ss);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += sums[j];
    store_from_f32<float, 4>(to, o, ss);
  });
}

// dx from the splits' sums.
template <typename T>
__global__ __launch_bounds__(kGatherRows* kWave) void lce_dx_join(const LceArgs a) {
  const LceInfo info = lce_info(a);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGatherRows + (threadIdx.x >> 6);
  if (row >= info.live) return;
  const int64_t t = load_one(a.rows + row, VBH_SPAN(a.rows, a.tokens));
  T* dx = static_cast<T*>(a.dx);
  const Span sd = VBH_SPAN(dx, a.tokens * a.hidden);
  const Span ss = VBH_SPAN(a.dx_sums, a.splits * a.tokens * a.padded);
  for (int64_t c = (threadIdx.x & (kWave - 1)) * 4; c < a.hidden; c += kWave * 4) {
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) {
      float v[4];
      load_f32<float, 4>(a.dx_sums + (s * a.tokens + row) * a.padded + c, v, ss);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = ldexpf(o[j], -info.shift);
    store_four(dx + t * a.hidden, c, a.hidden, o, sd);
  }
}

// dW where there are no tokens at all.
template <typename T>
__global__ __launch_bounds__(kGatherRows* kWave) void lce_zero(T* p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (kGatherRows * kWave) + threadIdx.x;
  if (i < n) store_one(p + i, static_cast<T>(0.0f), VBH_SPAN(p, n));
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

// Tiles, by size and type:
//   kBig   256 x 256 on 8 waves, one workgroup per CU: 16-bit products that fill the card with them
//   kMid   128 x 128 on 4 waves, two per CU: 0.85 of kBig's rate (8192 x 8192 x 8192: 1151 against
//          1375 TFLOP/s), in quarters of its portions; fp32 always, whose matrix instructions take
//          as long as the reads for either (125-134 TFLOP/s; the library's best 117-122)
//   kSmall 64 x 128, kTiny 32 x 128 on 4 waves: products of at most as many rows, whose time is
//          the read of W
enum Tile { kBig, kMid, kSmall, kTiny };
template <typename T, bool P_COLUMNS, bool Q_COLUMNS>
using BigTile = TileProduct<T, 256, 256, 4, 2, P_COLUMNS, Q_COLUMNS>;
template <typename T, bool P_COLUMNS, bool Q_COLUMNS>
using MidTile = TileProduct<T, 128, 128, 2, 2, P_COLUMNS, Q_COLUMNS>;
template <typename T, bool Q_COLUMNS>
using SmallTile = TileProduct<T, 64, 128, 1, 4, false, Q_COLUMNS>;
template <typename T, bool Q_COLUMNS>
using TinyTile = TileProduct<T, 32, 128, 1, 4, false, Q_COLUMNS>;

constexpr int64_t kPlainTokens = 64; // forward of at most these: no numbering of tokens
constexpr int64_t kPieceBytes = int64_t(256) << 20;
constexpr int64_t kPieceCols = 4096; // least of a piece
constexpr int64_t kMostPieceCols = int64_t(1) << 18;
constexpr int64_t kSplitCols = 1024; // least of a split of dx

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t tiles(int64_t n, int64_t each) { return (n + each - 1) / each; }
int value_bytes(int dt) { return dt == kF32 ? 4 : 2; }

// The tile of a product of `rows` (of P, whose lines have k contiguous unless P_COLUMNS) by `cols`.
Tile tile_of(int64_t rows, int64_t cols, int dt, bool p_columns = false) {
  if (!p_columns && rows <= 32) return kTiny;
  if (!p_columns && rows <= 64) return kSmall;
  if (dt == kF32) return kMid;
  // rounds of workgroups, by a round's time
  const int64_t big = tiles(tiles(rows, 256) * tiles(cols, 256), 256) * 100;
  const int64_t mid = tiles(tiles(rows, 128) * tiles(cols, 128), 512) * 59;
  return mid < big ? kMid : kBig;
}
int64_t tile_rows(Tile t) { return t == kBig ? 256 : t == kMid ? 128 : t == kSmall ? 64 : 32; }
int64_t tile_cols(Tile t) { return t == kBig ? 256 : 128; }
int64_t tile_fill(Tile t) { return t == kBig ? 256 : 512; }  // workgroups that fill the card

// f(TypeTag of the TileProduct)
template <typename T, bool Q_COLUMNS, typename F>
void with_tile(Tile t, F&& f) {
  switch (t) {
    case kBig:
      if constexpr (sizeof(T) == 2) f(TypeTag<BigTile<T, false, Q_COLUMNS>>{});
      break;
    case kMid: f(TypeTag<MidTile<T, false, Q_COLUMNS>>{}); break;
    case kSmall: f(TypeTag<SmallTile<T, Q_COLUMNS>>{}); break;
    case kTiny: f(TypeTag<TinyTile<T, Q_COLUMNS>>{}); break;
  }
}

// The workspace's parts, each at a multiple of 256 bytes.
struct LcePlan {
  int64_t padded = 0;
  int64_t pieces = 1, piece_cols = 0, pitch = 0;
  int64_t splits = 1, split_cols = 0;
  bool sums = false;
  Tile dx_tile = kBig;
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
    const int64_t n = tiles(vocab, tile_cols(tile_of(tokens, vocab, dt))) * tokens;
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
  const int64_t cols = std::min(p.piece_cols, vocab);  // of the first piece
  p.dx_tile = tile_of(tokens, hidden, dt);
  const int64_t out = tiles(tokens, tile_rows(p.dx_tile)) * tiles(hidden, tile_cols(p.dx_tile));
  p.splits = std::max<int64_t>(std::min(tiles(tile_fill(p.dx_tile), out), cols / kSplitCols), 1);
  p.split_cols = up(tiles(cols, p.splits), 128);
  p.splits = tiles(cols, p.split_cols);
  p.sums = p.splits > 1 || p.pieces > 1;
  if (p.sums) p.dx_sums = take(p.splits * tokens * p.padded * 4);
  return p;
}

template <typename T>
hipError_t forward(LceArgs a, int dt, bool number, hipStream_t s) {
  const unsigned tokens4 = static_cast<unsigned>(tiles(a.tokens, kGatherRows));
  hipError_t err = hipSuccess;
  auto done = [&] { return (err = hipGetLastError()) == hipSuccess; };
  if (number) {
    launch_kernel(lce_rows, dim3(1), dim3(kRowsLanes), 0, s, a);
    if (!done()) return err;
  }
  if (number || !a.x_direct) {
    launch_kernel(lce_gather<T>, dim3(tokens4), dim3(kGatherRows * kWave), 0, s, a);
    if (!done()) return err;
  }
  const Tile t = tile_of(a.tokens, a.vocab, dt);
  a.col_tiles = static_cast<int>(tiles(a.vocab, tile_cols(t)));
  with_tile<T, false>(t, [&](auto tag) {
    using G = typename decltype(tag)::type;
    const int64_t grid = tile_grid(tiles(a.tokens, G::BR), a.col_tiles);
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
  const unsigned tokens4 = static_cast<unsigned>(tiles(a.tokens, kGatherRows));
  hipError_t err = hipSuccess;
  auto done = [&] { return (err = hipGetLastError()) == hipSuccess; };
  launch_kernel(lce_rows, dim3(1), dim3(kRowsLanes), 0, s, a);
  if (!done()) return err;
  launch_kernel(lce_gather<T>, dim3(tokens4), dim3(kGatherRows * kWave), 0, s, a);
  if (!done()) return err;
  for (int64_t i = 0; i < p.pieces; ++i) {
    a.first = i * p.piece_cols;
    a.cols = std::min(p.piece_cols, a.vocab - a.first);
    a.pitch = up(a.cols, 16 / static_cast<int64_t>(sizeof(T)));
    const Tile t = tile_of(a.tokens, a.cols, dt);
    a.col_tiles = static_cast<int>(tiles(a.cols, tile_cols(t)));
    with_tile<T, false>(t, [&](auto tag) {
      using G = typename decltype(tag)::type;
      const int64_t grid = tile_grid(tiles(a.tokens, G::BR), a.col_tiles);
      launch_kernel(lce_dlogits<T, G>, dim3(static_cast<unsigned>(grid)), dim3(G::kLanes), 0, s, a);
    });
    if (!done()) return err;
    if (a.dw != nullptr) {
      auto go = [&](auto tag) {
        using G = typename decltype(tag)::type;
        const int64_t grid = tile_grid(tiles(a.cols, G::BR), tiles(a.hidden, G::BC));
        launch_kernel(lce_dweight<T, G>, dim3(static_cast<unsigned>(grid)), dim3(G::kLanes), 0, s,
                      a);
      };
      if constexpr (sizeof(T) == 2) {
        if (tile_of(a.cols, a.hidden, dt, true) == kBig) go(TypeTag<BigTile<T, true, true>>{});
        else go(TypeTag<MidTile<T, true, true>>{});
      } else {
        go(TypeTag<MidTile<T, true, true>>{});
      }
      if (!done()) return err;
    }
    if (a.dx == nullptr) continue;
    with_tile<T, true>(p.dx_tile, [&](auto tag) {
      using G = typename decltype(tag)::type;
      const int64_t grid = tile_grid(tiles(a.tokens, G::BR), tiles(a.hidden, G::BC));
      // a shorter last piece may have fewer splits: those before it have summed into all
      launch_kernel(lce_dx<T, G>,
                    dim3(static_cast<unsigned>(grid),
                         static_cast<unsigned>(tiles(a.cols, a.split_cols))),
                    dim3(G::kLanes), 0, s, a, i > 0 ? 1 : 0);
    });
    if (!done()) return err;
  }
  if (a.dx != nullptr && p.sums) {
    launch_kernel(lce_dx_join<T>, dim3(tokens4), dim3(kGatherRows * kWave), 0, s, a);
    done();
  }
  return err;
}

}  // namespace

int64_t linear_ce_workspace_bytes(int64_t tokens, int64_t hidden, int64_t vocab, int dt,
                                  bool pad_weight, bool backward) {
  return lce_plan(tokens, hidden, vocab, dt, pad_weight, backward).bytes;
}

hipError_t launch_linear_ce(LceArgs a, int dt, bool back, void* workspace, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (a.tokens == 0) {
    dispatch_float_type(dt, [&](auto tag) {
      using T = typename decltype(tag)::type;
      const int64_t n = a.vocab * a.hidden;
      launch_kernel(lce_zero<T>, dim3(static_cast<unsigned>(tiles(n, kGatherRows * kWave))),
                    dim3(kGatherRows * kWave), 0, s, static_cast<T*>(a.dw), n);
      err = hipGetLastError();
    });
    return err;
  }
  const bool pad_weight = a.w == nullptr;
  const LcePlan p = lce_plan(a.tokens, a.hidden, a.vocab, dt, pad_weight, back);
  char* ws = static_cast<char*>(workspace);
  a.padded = p.padded;
  a.x_packed = ws + p.x;
  const bool number = back || a.tokens > kPlainTokens;
  if (number) {
    a.info = ws + p.info;
    a.rows = reinterpret_cast<int*>(ws + p.rows);
    a.place = reinterpret_cast<int*>(ws + p.place);
  }
  if (back) {
    a.piece = ws + p.piece;
    a.splits = static_cast<int>(p.splits);
    a.split_cols = p.split_cols;
    if (p.sums) a.dx_sums = reinterpret_cast<float*>(ws + p.dx_sums);
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
