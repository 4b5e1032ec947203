// Gradients of LayerNorm and RMSNorm over the last axis, for gfx950.  With m the row's
// mean (RMSNorm: 0), d = x - m, r = 1 / sqrt(mean(d^2) + eps), u = d r, g = dy w:
//
//   dx = r (g - mean(g) - u mean(g u))     (RMSNorm: without mean(g))
//   dw = sum over rows of dy u,  db = sum over rows of dy
//
// m and r are formed again from the row, which is read anyway: the forward keeps
// nothing for the backward.  A row is owned by a group of lanes and held in registers
// in its storage type, x and dy are read once and dx is written once.  A workgroup
// walks over rows with the next row's loads in flight, its lanes keep the fp32 sums
// of their columns' dw and db, and its groups' sums are added through the LDS at the
// end into one row of `parts`; a second kernel adds the rows of parts.  All in a fixed
// order.
#include <algorithm>

#include "vbh_launch.h"

namespace vbh {

namespace {

// A lane's accesses of a row: vector i begins at column at[i]; its first skip[i] values
// belong to the vector before it (the last vector of a row that is no whole number of
// vectors is moved back to end with it), all V where the lane has no i-th vector.
template <int V, int IT>
struct NormLane {
  int at[IT], skip[IT];
  __device__ __forceinline__ NormLane(int g, int tpr, int cols) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int first = (g + i * tpr) * V;
      at[i] = first + V <= cols ? first : cols - V;
      skip[i] = min(first - at[i], V);
    }
  }
};

// Sums of N values over a row's lanes, in every lane.  Each call of a kernel instance
// between two barriers needs a buffer of its own.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int tpr, float (*lds)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_allreduce<Sum>(v[i], tpr < kWave ? tpr : kWave);
  if (tpr <= kWave) return;
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int nwaves = tpr >> 6;
  const int first = first_wave_of_group(wave, nwaves, tpr);
  if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) lds[wave][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lds[first][i];
  for (int w = 1; w < nwaves; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += lds[first + w][i];
  }
}

struct NormBuffers {  // of two rows in turn
  float mean[2][kMaxWaves][1], dots[2][kMaxWaves][3], again[2][kMaxWaves][1];
};

__device__ __forceinline__ bool out_of_range(float v) { return !(__builtin_fabsf(v) <= 0x1p127f); }

// The workgroup's rows.  dw, db: the lane's sums.  True where the gradients of a row of
// the lane's group need sum(g u), which has to wait for r, as sum(g d) leaves the range
// of 32 bits or may lose terms below 2^-149 (r past 2^20, where eps is next to nothing).
// AGAIN goes over the rows once more and stores those rows' dx.
template <typename T, typename W, int V, int IT, bool LN, bool RAGGED, bool AGAIN>
__device__ __forceinline__ bool norm_rows(const NormGradArgs& a, NormBuffers& lds,
                                          float (&dw)[IT][V], float (&db)[IT][V]) {
  typedef typename Raw<T, V>::type R;
  const GroupShape gs = group_shape(a.tpr);
  const NormLane<V, IT> l(gs.g, a.tpr, a.cols);
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  const Span sx = VBH_SPAN(x, a.rows * a.cols), sg = VBH_SPAN(dy, a.rows * a.cols);
  const Span sy = VBH_SPAN(static_cast<T*>(a.dx), a.rows * a.cols);
  const Span sw = VBH_SPAN(static_cast<const W*>(a.w), a.cols);
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  float w[IT][V];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    if constexpr (sizeof(W) == sizeof(T)) {
      const auto raw = load_any<W, V, false>(static_cast<const W*>(a.w) + l.at[i], sw);
#pragma unroll
      for (int k = 0; k < V; ++k) w[i][k] = raw_at<W, V>(raw, k);
    } else {  // fp32 weights of 16-bit rows, in two halves
      constexpr int H = V > 1 ? V / 2 : 1;
#pragma unroll
      for (int h = 0; h < V / H; ++h) {
        const auto raw = load_any<W, H, false>(static_cast<const W*>(a.w) + l.at[i] + h * H, sw);
#pragma unroll
        for (int k = 0; k < H; ++k) w[i][h * H + k] = raw_at<W, H>(raw, k);
      }
    }
  }
  // value k of vector i counts
  auto counts = [&](int i, int k) { return RAGGED ? k >= l.skip[i] : l.skip[i] == 0; };

  const int64_t step = static_cast<int64_t>(gridDim.x) * gs.per_block;
  int64_t row = static_cast<int64_t>(blockIdx.x) * gs.per_block + gs.sub;
  // every group makes as many turns as the workgroup's first (barriers); in turns past
  // the last row it works on row 0 again, and nothing of it counts
  const int64_t base = static_cast<int64_t>(blockIdx.x) * gs.per_block;
  const int64_t turns = base < a.rows ? (a.rows - base + step - 1) / step : 0;
  bool again = false;
  R xr[IT], gr[IT];
  auto load = [&](int64_t to, R (&xs)[IT], R (&gr2)[IT]) {
    const int64_t at = (to < a.rows ? to : 0) * a.cols;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      xs[i] = load_any<T, V, true>(x + at + l.at[i], sx);
      gr2[i] = load_any<T, V, true>(dy + at + l.at[i], sg);
    }
  };
  if (turns > 0) load(row, xr, gr);
  for (int64_t turn = 0; turn < turns; ++turn, row += step) {
    const bool live = row < a.rows;
    const int buf = static_cast<int>(turn & 1);
    R xn[IT], gn[IT];
    if (turn + 1 < turns) load(row + step, xn, gn);
    float m = 0.0f;
    if constexpr (LN) {
      float sum[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        float part = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = raw_at<T, V>(xr[i], k);
          part += RAGGED && !counts(i, k) ? 0.0f : v;
        }
        sum[0] += RAGGED || counts(i, 0) ? part : 0.0f;
      }
      row_sums<1>(sum, a.tpr, lds.mean[buf]);
      m = sum[0] * inv_n;
      reload_barrier<T, V, IT>(xr);
    }
    float dots[3] = {0.0f, 0.0f, 0.0f};  // d^2, g d, g
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float part[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const bool ok = !RAGGED || counts(i, k);
        const float d = ok ? raw_at<T, V>(xr[i], k) - m : 0.0f;
        const float g = ok ? raw_at<T, V>(gr[i], k) * w[i][k] : 0.0f;
        part[0] = fmaf(d, d, part[0]);
        part[1] = fmaf(g, d, part[1]);
        if (LN) part[2] += g;
      }
#pragma unroll
      for (int j = 0; j < 3; ++j) dots[j] += RAGGED || counts(i, 0) ? part[j] : 0.0f;
    }
    row_sums<3>(dots, a.tpr, lds.dots[buf]);
    reload_barrier<T, V, IT>(xr);
    reload_barrier<T, V, IT>(gr);
    const float r = 1.0f / __builtin_sqrtf(fmaf(dots[0], inv_n, a.eps));
    const bool needs = live && (out_of_range(dots[1]) || r > 0x1p20f);
    again = again || needs;
    float mean_gu = dots[1] * r * inv_n;
    if constexpr (AGAIN) {
      float dot[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < IT; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float u = (raw_at<T, V>(xr[i], k) - m) * r;
          dot[0] += counts(i, k) ? raw_at<T, V>(gr[i], k) * w[i][k] * u : 0.0f;
        }
      }
      row_sums<1>(dot, a.tpr, lds.again[buf]);
      mean_gu = dot[0] * inv_n;
    }
    const float mean_g = dots[2] * inv_n;
    T* out = static_cast<T*>(a.dx) + (live ? row : 0) * a.cols;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float u = (raw_at<T, V>(xr[i], k) - m) * r;
        const float gy = raw_at<T, V>(gr[i], k);
        // r last: g r may leave the range of 32 bits
        o[k] = r * (fmaf(gy, w[i][k], -mean_g) - u * mean_gu);
        if constexpr (!AGAIN) {
          // sums of values that do not count are not written: only rows that are not
          // the group's have to stay out
          dw[i][k] = live ? fmaf(gy, u, dw[i][k]) : dw[i][k];
          if (LN) db[i][k] = live ? db[i][k] + gy : db[i][k];
        }
      }
      if (AGAIN ? !needs : !live) continue;
      if (l.skip[i] == 0) {
        store_any<T, V, true>(out + l.at[i], o, sy);
      } else if constexpr (RAGGED) {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (counts(i, k)) store_any<T, 1, true>(out + l.at[i] + k, o + k, sy);
      }
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      xr[i] = xn[i];
      gr[i] = gn[i];
    }
  }
  return again;
}

// Lanes of a wave that hold the same columns (groups of tpr < 64 lanes) added up.
template <int V, int IT>
__device__ __forceinline__ void add_groups(float (&v)[IT][V], int tpr) {
#pragma unroll
  for (int i = 0; i < IT; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      for (int s = tpr; s < kWave; s *= 2) v[i][k] += __shfl_xor(v[i][k], s);
    }
  }
}

// The workgroup's sums of one vector into its row of parts, group after group.
template <int V, int IT>
__device__ __forceinline__ void write_sums(const NormGradArgs& a, const float (&v)[IT][V],
                                           float* sums, int64_t row) {
  const int tpr = max(a.tpr, kWave);  // a wave's groups are one by now
  const GroupShape gs = group_shape(tpr);
  const NormLane<V, IT> l(gs.g & (a.tpr - 1), a.tpr, a.cols);
  const NormLane<V, IT> lane = a.tpr < kWave ? l : NormLane<V, IT>(gs.g, a.tpr, a.cols);
  const bool owner = a.tpr >= kWave || gs.g < a.tpr;
  for (int q = 0; q < gs.per_block; ++q) {
    if (owner && gs.sub == q) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if (k < lane.skip[i]) continue;
          float* to = sums + lane.at[i] + k;
          *to = q == 0 ? v[i][k] : *to + v[i][k];
        }
      }
    }
    __syncthreads();
  }
  float* out = a.parts + row * a.pitch;
  const Span sp = VBH_SPAN(a.parts, a.part_rows * a.pitch);
  for (int c = static_cast<int>(threadIdx.x); c < a.cols; c += static_cast<int>(blockDim.x))
    store_any<float, 1, false>(out + c, sums + c, sp);
  __syncthreads();
}

template <typename T, typename W, int V, int IT, bool LN, bool RAGGED, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_grads(const NormGradArgs a) {
  extern __shared__ __align__(16) float norm_sums[];
  __shared__ NormBuffers lds;
  float dw[IT][V], db[IT][V];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.0f;
  }
  const bool again = norm_rows<T, W, V, IT, LN, RAGGED, false>(a, lds, dw, db);
  if (__builtin_expect(__syncthreads_or(again), 0))
    norm_rows<T, W, V, IT, LN, RAGGED, true>(a, lds, dw, db);
  if (a.parts == nullptr) return;
  add_groups<V, IT>(dw, a.tpr);
  write_sums<V, IT>(a, dw, norm_sums, blockIdx.x);
  if constexpr (LN) {
    add_groups<V, IT>(db, a.tpr);
    write_sums<V, IT>(a, db, norm_sums, gridDim.x + blockIdx.x);
  }
}

// ---------------------------------------------------------------------------
// rows beyond the registers: the row's statistics first, then tiles of columns that
// read x and dy once more
// ---------------------------------------------------------------------------

constexpr int kWideLanes = 256;

struct WideStat {
  float m, r, mean_g, mean_gu;
};

// One workgroup per row, value by value in three passes over the row (the second and
// third from the L2).
template <typename T, typename W, bool LN>
__global__ __launch_bounds__(kMaxBlock) void norm_wide_stats(const NormGradArgs a, float* stats) {
  __shared__ float mean[kMaxWaves][1], squares[kMaxWaves][1], dots[kMaxWaves][2];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.cols;
  const T* dy = static_cast<const T*>(a.dy) + row * a.cols;
  const W* w = static_cast<const W*>(a.w);
  const Span sx = VBH_SPAN(x, a.cols), sg = VBH_SPAN(dy, a.cols), sw = VBH_SPAN(w, a.cols);
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  const int first = static_cast<int>(threadIdx.x), block = static_cast<int>(blockDim.x);
  WideStat s{0.0f, 0.0f, 0.0f, 0.0f};
  auto at = [](const auto* p, int64_t c, const Span& sp) {
    float v;
    load_f32<std::decay_t<decltype(*p)>, 1>(p + c, &v, sp);
    return v;
  };
  if constexpr (LN) {
    float sum[1] = {0.0f};
    for (int64_t c = first; c < a.cols; c += block) sum[0] += at(x, c, sx);
    row_sums<1>(sum, block, mean);
    s.m = sum[0] * inv_n;
  }
  float sq[1] = {0.0f};
  for (int64_t c = first; c < a.cols; c += block) {
    const float d = at(x, c, sx) - s.m;
    sq[0] = fmaf(d, d, sq[0]);
  }
  row_sums<1>(sq, block, squares);
  s.r = 1.0f / __builtin_sqrtf(fmaf(sq[0], inv_n, a.eps));
  float dot[2] = {0.0f, 0.0f};
  for (int64_t c = first; c < a.cols; c += block) {
    const float g = at(dy, c, sg) * at(w, c, sw);
    dot[0] = fmaf(g, (at(x, c, sx) - s.m) * s.r, dot[0]);
    if (LN) dot[1] += g;
  }
  row_sums<2>(dot, block, dots);
  if (threadIdx.x == 0) {
    const float o[4] = {s.m, s.r, dot[1] * inv_n, dot[0] * inv_n};
    store_any<float, 4, false>(stats + row * 4, o, VBH_SPAN(stats, a.rows * 4));
  }
}

// A workgroup: kWideLanes columns of every gridDim.y-th row.
template <typename T, typename W, bool LN>
__global__ __launch_bounds__(kWideLanes) void norm_wide_apply(const NormGradArgs a,
                                                             const float* stats) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kWideLanes + threadIdx.x;
  if (c >= a.cols) return;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  const Span sx = VBH_SPAN(x, a.rows * a.cols), sg = VBH_SPAN(dy, a.rows * a.cols);
  const Span sy = VBH_SPAN(static_cast<T*>(a.dx), a.rows * a.cols);
  const Span st = VBH_SPAN(stats, a.rows * 4);
  float w, dw = 0.0f, db = 0.0f;
  load_f32<W, 1>(static_cast<const W*>(a.w) + c, &w, VBH_SPAN(static_cast<const W*>(a.w), a.cols));
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float xv, gy, s[4];
    load_f32<T, 1>(x + row * a.cols + c, &xv, sx);
    load_f32<T, 1>(dy + row * a.cols + c, &gy, sg);
    load_f32<float, 4>(stats + row * 4, s, st);
    const float u = (xv - s[0]) * s[1];
    const float o = s[1] * (fmaf(gy, w, -s[2]) - u * s[3]);
    store_any<T, 1, true>(static_cast<T*>(a.dx) + row * a.cols + c, &o, sy);
    dw = fmaf(gy, u, dw);
    db += gy;
  }
  if (a.parts == nullptr) return;
  const Span sp = VBH_SPAN(a.parts, a.part_rows * a.pitch);
  store_any<float, 1, false>(a.parts + blockIdx.y * a.pitch + c, &dw, sp);
  if constexpr (LN)
    store_any<float, 1, false>(a.parts + (gridDim.y + blockIdx.y) * a.pitch + c, &db, sp);
}

// ---------------------------------------------------------------------------
// sums over the rows of parts
// ---------------------------------------------------------------------------

// A workgroup: 16 columns of one vector, four to a lane and 256 lines of lanes, so that
// 256 rows take one round of loads.  Lines are added up through the wave, waves through
// the LDS, in order.
constexpr int kPartCols = 16;
constexpr int kPartLanes = 1024;

template <typename W>
__global__ __launch_bounds__(kPartLanes) void norm_weight_grads(const float* parts, int rows,
                                                                int64_t pitch, int64_t cols,
                                                                W* dw, W* db) {
  __shared__ float sums[kPartLanes / kWave][kPartCols];
  W* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  const Span sp = VBH_SPAN(parts, static_cast<int64_t>(rows) * gridDim.y * pitch);
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kPartCols;
  const int line = wave * 16 + lane / 4;
  const float* from = parts + blockIdx.y * static_cast<int64_t>(rows) * pitch + col + (lane & 3) * 4;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (col + (lane & 3) * 4 < pitch) {
    for (int r = line; r < rows; r += kPartLanes / 4) {
      float x[4];
      load_f32<float, 4>(from + r * pitch, x, sp);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int s = 4; s < kWave; s *= 2) v[i] += __shfl_xor(v[i], s);
  }
  if (lane < 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][lane * 4 + i] = v[i];
  }
  __syncthreads();
  const int c = static_cast<int>(threadIdx.x);
  if (c >= kPartCols || col + c >= cols) return;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kPartLanes / kWave; ++i) sum += sums[i][c];
  store_any<W, 1, false>(out + col + c, &sum, VBH_SPAN(out, cols));
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

constexpr int kNormMaxIt = 4;
constexpr int64_t kNormCus = 256;

// How a launch is laid out, a function of its sizes and types alone.
struct NormShape {
  bool wide = false;
  int v = 1, it = 1, tpr = 64, block = 256;
  int64_t grid = 0;  // rows of parts for each vector
};

NormShape norm_shape(int64_t rows, int64_t cols, int dt) {
  NormShape s;
  const int vn = dt == kF32 ? 4 : 8;
  s.v = cols >= vn ? vn : 1;
  const int64_t nvec = (cols + s.v - 1) / s.v;
  if (nvec > int64_t(kNormMaxIt) * kMaxBlock) {
    s.wide = true;
    s.grid = std::max<int64_t>(std::min<int64_t>(rows, 64), 1);
    return s;
  }
  if (nvec <= kWave) {
    s.tpr = 1;
    while (s.tpr < nvec) s.tpr *= 2;
  } else if (nvec <= int64_t(kNormMaxIt) * kWave) {
    s.it = static_cast<int>((nvec + kWave - 1) / kWave);
  } else {
    s.it = nvec <= 2 * kMaxBlock ? 2 : static_cast<int>((nvec + kMaxBlock - 1) / kMaxBlock);
    s.tpr = static_cast<int>((nvec + int64_t(s.it) * kWave - 1) / (int64_t(s.it) * kWave)) * kWave;
  }
  // as many groups to a workgroup as leave every CU one
  const int most = s.it > 2 ? 512 : 1024;
  s.block = std::max(s.tpr, 256 / s.tpr * s.tpr);
  while (s.block + s.tpr <= most && rows >= kNormCus * (s.block / s.tpr + 1)) s.block += s.tpr;
  if (s.tpr < kWave) s.block = std::max(s.block / kWave * kWave, kWave);
  const int64_t per = s.block / s.tpr;
  s.grid = std::max<int64_t>(std::min<int64_t>((rows + per - 1) / per, kNormCus), 1);
  return s;
}

int64_t norm_pitch(int64_t cols) { return (cols + 3) / 4 * 4; }

template <typename T, typename W, bool LN>
hipError_t launch_norm(NormGradArgs a, const NormShape& s, float* stats, hipStream_t stream) {
  hipError_t err = hipSuccess;
  if (s.wide) {
    launch_kernel(norm_wide_stats<T, W, LN>, dim3(static_cast<unsigned>(a.rows)), dim3(kMaxBlock),
                  0, stream, a, stats);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    const unsigned tiles = static_cast<unsigned>((a.cols + kWideLanes - 1) / kWideLanes);
    launch_kernel(norm_wide_apply<T, W, LN>, dim3(tiles, static_cast<unsigned>(s.grid)),
                  dim3(kWideLanes), 0, stream, a, stats);
    return hipGetLastError();
  }
  a.tpr = s.tpr;
  auto go = [&](auto kernel) {
    const unsigned bytes = a.parts != nullptr ? static_cast<unsigned>(a.cols * sizeof(float)) : 0;
    launch_kernel(kernel, dim3(static_cast<unsigned>(s.grid)), dim3(s.block), bytes, stream, a);
    err = hipGetLastError();
  };
  constexpr int VN = Vec<T>::n;
  dispatch_bool(s.v > 1 && a.cols % VN != 0, [&](auto rc) {
    constexpr bool RAGGED = decltype(rc)::value;
    auto by_it = [&](auto ic) {
      constexpr int IT = decltype(ic)::value;
      if (IT > 2 && s.block <= 512) go(norm_grads<T, W, VN, IT, LN, RAGGED, IT <= 2 ? 1024 : 512>);
      else go(norm_grads<T, W, VN, IT, LN, RAGGED, 1024>);
    };
    if (s.v == 1) go(norm_grads<T, W, 1, 1, LN, false, 1024>);
    else if (s.it == 1) by_it(std::integral_constant<int, 1>{});
    else if (s.it == 2) by_it(std::integral_constant<int, 2>{});
    else if (s.it == 3) by_it(std::integral_constant<int, 3>{});
    else by_it(std::integral_constant<int, 4>{});
  });
  return err;
}

}  // namespace

int64_t norm_bwd_workspace_floats(int64_t rows, int64_t cols, int dt, bool ln) {
  const NormShape s = norm_shape(rows, cols, dt);
  return (ln ? 2 : 1) * s.grid * norm_pitch(cols) + (s.wide ? 4 * rows : 0);
}

bool norm_bwd_needs_workspace(int64_t rows, int64_t cols, int dt, bool sums) {
  return sums || norm_shape(rows, cols, dt).wide;
}

hipError_t launch_norm_bwd(NormGradArgs a, bool ln, int dt, int wdt, void* dw, void* db,
                           float* workspace, hipStream_t stream) {
  const NormShape s = norm_shape(a.rows, a.cols, dt);
  const bool sums = dw != nullptr || db != nullptr;
  a.pitch = norm_pitch(a.cols);
  a.part_rows = (ln ? 2 : 1) * s.grid;
  a.parts = sums ? workspace : nullptr;
  float* stats = workspace + a.part_rows * a.pitch;
  hipError_t err = hipSuccess;
  if (a.rows > 0) {
    dispatch_float_type(dt, [&](auto tt) {
      using T = typename decltype(tt)::type;
      dispatch_bool(ln, [&](auto lc) {
        constexpr bool LN = decltype(lc)::value;
        if (wdt == kF32) err = launch_norm<T, float, LN>(a, s, stats, stream);
        else err = launch_norm<T, T, LN>(a, s, stats, stream);
      });
    });
  }
  if (err != hipSuccess || !sums) return err;
  auto sum = [&](auto tag) {
    using W = typename decltype(tag)::type;
    launch_kernel(norm_weight_grads<W>,
                  dim3(static_cast<unsigned>((a.cols + kPartCols - 1) / kPartCols), ln ? 2 : 1),
                  dim3(kPartLanes), 0, stream, static_cast<const float*>(a.parts),
                  a.rows > 0 ? static_cast<int>(s.grid) : 0, a.pitch, a.cols,
                  static_cast<W*>(dw), static_cast<W*>(db));
    err = hipGetLastError();
  };
  if (wdt == kF32) sum(TypeTag<float>{});
  else dispatch_float_type(dt, sum);
  return err;
}

}  // namespace vbh
