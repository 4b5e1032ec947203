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
// order.  Rows of more than 4096 16-byte vectors do not fit: their x is read four times and
// dy twice (norm_wide_stats, norm_wide_apply).
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

// What a row is reduced to: its mean (RMSNorm: 0), and with d = x - mean the sums of d^2, g d
// and g.
struct RowDots {
  float m, dd, gd, g;
};
struct NormBuffers {  // of two rows in turn
  RowDots dots[2][kMaxWaves];
  float again[2][kMaxWaves][1];
  float counts[kMaxWaves];  // LayerNorm: values that each wave has of a row
};

// `mine`: the dots of the lane's wave (tpr <= 64: of its group, and the row's already) about that
// wave's own mean.  Those of the row: with M the mean of the waves' means m_w by their counts n_w,
// d^2 grows by n_w (m_w - M)^2 and g d by (m_w - M) g_w.  One barrier a row where sums about the
// row's mean would take two.
template <bool LN>
__device__ __forceinline__ RowDots row_dots(RowDots mine, int tpr, float inv_n, RowDots* dots,
                                            const float* counts) {
  if (tpr <= kWave) return mine;
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int nwaves = tpr >> 6;
  const int first = first_wave_of_group(wave, nwaves, tpr);
  if ((threadIdx.x & (kWave - 1)) == 0) dots[wave] = mine;
  __syncthreads();
  RowDots all{0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (LN) {
    for (int w = 0; w < nwaves; ++w) all.m = fmaf(dots[first + w].m, counts[first + w], all.m);
    all.m *= inv_n;
  }
  for (int w = 0; w < nwaves; ++w) {
    const RowDots o = dots[first + w];
    const float off = LN ? o.m - all.m : 0.0f;
    all.dd += LN ? fmaf(off * off, counts[first + w], o.dd) : o.dd;
    all.gd += LN ? fmaf(off, o.g, o.gd) : o.gd;
    all.g += o.g;
  }
  return all;
}

__device__ __forceinline__ bool out_of_range(float v) { return !(__builtin_fabsf(v) <= 0x1p127f); }

// V weights in their storage type.
template <typename W, int V> struct NormWeights {
  static constexpr int kPart = V * static_cast<int>(sizeof(W)) > 16 ? V / 2 : V;  // one access
  typename Raw<W, kPart>::type part[V / kPart];
  __device__ __forceinline__ void load(const W* w, const Span& s) {
#pragma unroll
    for (int i = 0; i < V / kPart; ++i) part[i] = load_any<W, kPart, false>(w + i * kPart, s);
  }
  __device__ __forceinline__ float at(int k) const {
    return raw_at<W, kPart>(part[k / kPart], k % kPart);
  }
  // keeps 16-bit weights as they are from row to row, instead of their widened values
  __device__ __forceinline__ void keep() { reload_barrier<W, kPart, V / kPart>(part); }
};

// The lane's fp32 sums of dw and db.
template <int V, int IT> struct NormSums {
  float dw[IT][V], db[IT][V];
};

// The workgroup's rows.  True where the gradients of a row of the lane's group need sum(g u),
// which has to wait for r, as sum(g d) leaves the range of 32 bits or may lose terms below 2^-149
// (r past 2^20, where eps is next to nothing).  AGAIN goes over the rows once more and stores
// those rows' dx.
//
// The next row's loads are in flight while a row is worked on: in registers, or (AHEAD, where a
// lane has more than two whole vectors of a row) straight into the LDS, each wave's in its own part
// without a barrier.  There a wave counts what it has to wait for: its loads and stores complete in
// order, and behind a row's loads come the IT stores of the row before, whatever its lanes have of
// that (buffer stores, of which those beyond the resource's range are dropped).  (With two vectors a
// lane, one or two rows ahead in the LDS are slower: 8192 x 4096 bf16 LayerNorm 52.3 and 50.5 us, in
// registers 46.9.)
template <typename T, typename W, int V, int IT, bool LN, bool RAGGED, bool AHEAD, bool AGAIN>
__device__ __forceinline__ bool norm_rows(const NormGradArgs& a, NormBuffers& lds, char* slot,
                                          NormSums<V, IT>& sums) {
  typedef typename Raw<T, V>::type R;
  const GroupShape gs = group_shape(a.tpr);
  const NormLane<V, IT> l(gs.g, a.tpr, a.cols);
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  const Span sx = VBH_SPAN(x, a.rows * a.cols), sg = VBH_SPAN(dy, a.rows * a.cols);
  const Span sy = VBH_SPAN(static_cast<T*>(a.dx), a.rows * a.cols);
  const Span sw = VBH_SPAN(static_cast<const W*>(a.w), a.cols);
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  // lanes with several vectors of a row share it with their whole wave
  constexpr bool kWaveRow = IT > 1;
  const int width = kWaveRow || a.tpr > kWave ? kWave : a.tpr;
  // value k of vector i counts
  auto counts = [&](int i, int k) { return RAGGED ? k >= l.skip[i] : l.skip[i] == 0; };

  const int64_t step = static_cast<int64_t>(gridDim.x) * gs.per_block;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * gs.per_block;
  // every group makes as many turns as the workgroup's first (barriers); in turns past
  // the last row it works on row 0 again, and nothing of it counts
  const int64_t turns = base < a.rows ? (a.rows - base + step - 1) / step : 0;
  int64_t row = base + (kWaveRow ? __builtin_amdgcn_readfirstlane(gs.sub) : gs.sub);
  bool again = false;
  R xr[IT], gr[IT], xn[AHEAD ? 1 : IT], gn[AHEAD ? 1 : IT];
  auto load = [&](int64_t to, R* xs, R* gs_) {
    const int64_t at = (to < a.rows ? to : 0) * a.cols;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (a.nt) {
        xs[i] = load_any<T, V, true>(x + at + l.at[i], sx);
        gs_[i] = load_any<T, V, true>(dy + at + l.at[i], sg);
      } else {
        xs[i] = load_any<T, V, false>(x + at + l.at[i], sx);
        gs_[i] = load_any<T, V, false>(dy + at + l.at[i], sg);
      }
    }
  };
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  auto place = [&](int j) { return slot + (wave * 2 * IT + j) * kWave * 16; };  // j-th access
  auto stage = [&](int64_t to) {
    if constexpr (AHEAD) {
      const int64_t at = (to < a.rows ? to : 0) * a.cols;
      typedef __attribute__((address_space(1))) const void global_void;
      typedef __attribute__((address_space(3))) void lds_void;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const T* px = x + at + l.at[i];
        const T* pg = dy + at + l.at[i];
        if (VBH_IN_SPAN(sx, px, 16))
          __builtin_amdgcn_global_load_lds((global_void*)px, (lds_void*)place(2 * i), 16, 0, 2);
        if (VBH_IN_SPAN(sg, pg, 16))
          __builtin_amdgcn_global_load_lds((global_void*)pg, (lds_void*)place(2 * i + 1), 16, 0,
                                           2);
      }
    }
  };
  if (turns > 0) {
    if constexpr (AHEAD) {
      stage(row);
    } else {
      load(row, xr, gr);
    }
  }
  NormWeights<W, V> w[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) w[i].load(static_cast<const W*>(a.w) + l.at[i], sw);
  // LayerNorm: values of a row that the lane's wave (tpr < 64: group) holds
  float inv_mine = 0.0f;
  if constexpr (LN) {
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < IT; ++i) mine += static_cast<float>(RAGGED ? V - l.skip[i] : counts(i, 0) * V);
    mine = wave_allreduce<Sum>(mine, width);
    if (lane == 0) lds.counts[wave] = mine;
    inv_mine = mine > 0.0f ? 1.0f / mine : 0.0f;
  }

  for (int64_t turn = 0; turn < turns; ++turn, row += step) {
    // (AHEAD: one row to a workgroup.  A constant saves two selects per value: 2048 rows of 20480 bf16
    // values, LayerNorm, 68.3 us against 72.9)
    const bool live = AHEAD || row < a.rows;
    const int buf = static_cast<int>(turn & 1);
    if constexpr (AHEAD) {
      if (turn == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IT) : "memory");
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        xr[i] = *reinterpret_cast<const R*>(place(2 * i) + lane * 16);
        gr[i] = *reinterpret_cast<const R*>(place(2 * i + 1) + lane * 16);
      }
      // read before the next row's loads write there
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (turn + 1 < turns) stage(row + step);
    } else {
      if (turn + 1 < turns) load(row + step, xn, gn);
    }
    if constexpr (IT > 2) {
#pragma unroll
      for (int i = 0; i < IT; ++i) w[i].keep();
    }
    RowDots dots{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (LN) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        float part = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = raw_at<T, V>(xr[i], k);
          part += RAGGED && !counts(i, k) ? 0.0f : v;
        }
        dots.m += RAGGED || counts(i, 0) ? part : 0.0f;
      }
      dots.m = wave_allreduce<Sum>(dots.m, width) * inv_mine;
      reload_barrier<T, V, IT>(xr);
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float part[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const bool ok = !RAGGED || counts(i, k);
        const float d = ok ? raw_at<T, V>(xr[i], k) - dots.m : 0.0f;
        const float g = ok ? raw_at<T, V>(gr[i], k) * w[i].at(k) : 0.0f;
        part[0] = fmaf(d, d, part[0]);
        part[1] = fmaf(g, d, part[1]);
        if (LN) part[2] += g;
      }
      const bool ok = RAGGED || counts(i, 0);
      dots.dd += ok ? part[0] : 0.0f;
      dots.gd += ok ? part[1] : 0.0f;
      if (LN) dots.g += ok ? part[2] : 0.0f;
    }
    dots.dd = wave_allreduce<Sum>(dots.dd, width);
    dots.gd = wave_allreduce<Sum>(dots.gd, width);
    if constexpr (LN) dots.g = wave_allreduce<Sum>(dots.g, width);
    dots = row_dots<LN>(dots, a.tpr, inv_n, lds.dots[buf], lds.counts);
    reload_barrier<T, V, IT>(xr);
    reload_barrier<T, V, IT>(gr);
    const float r = 1.0f / __builtin_sqrtf(fmaf(dots.dd, inv_n, a.eps));
    const bool needs = live && (out_of_range(dots.gd) || r > 0x1p20f);
    again = again || needs;
    float mean_gu = dots.gd * r * inv_n;
    if constexpr (AGAIN) {
      float dot[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < IT; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float u = (raw_at<T, V>(xr[i], k) - dots.m) * r;
          dot[0] += counts(i, k) ? raw_at<T, V>(gr[i], k) * w[i].at(k) * u : 0.0f;
        }
      }
      row_sums<1>(dot, a.tpr, lds.again[buf]);
      mean_gu = dot[0] * inv_n;
    }
    const float mean_g = dots.g * inv_n;
    T* out = static_cast<T*>(a.dx) + (live ? row : 0) * a.cols;
    // staged: the workgroup's rows of this turn
    const int64_t at0 = (base + turn * step) * a.cols;
    const int64_t left = (a.rows * a.cols - at0) * static_cast<int64_t>(sizeof(T));
    __amdgpu_buffer_rsrc_t rsrc;
    if constexpr (AHEAD)
      rsrc = __builtin_amdgcn_make_buffer_rsrc(
          static_cast<T*>(a.dx) + at0, static_cast<short>(0),
          __builtin_amdgcn_readfirstlane(static_cast<int>(left < 0x40000000 ? left : 0x40000000)),
          kRawBufferWord3);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float u = (raw_at<T, V>(xr[i], k) - dots.m) * r;
        const float gy = raw_at<T, V>(gr[i], k);
        // r last: g r may leave the range of 32 bits
        o[k] = r * (fmaf(gy, w[i].at(k), -mean_g) - u * mean_gu);
        if constexpr (!AGAIN) {
          // sums of values that do not count are not written: only rows that are not
          // the group's have to stay out
          sums.dw[i][k] = live ? fmaf(gy, u, sums.dw[i][k]) : sums.dw[i][k];
          if (LN) sums.db[i][k] = live ? sums.db[i][k] + gy : sums.db[i][k];
        }
      }
      if constexpr (AHEAD) {
        typedef int i32x4 __attribute__((ext_vector_type(4)));
        R res;
#pragma unroll
        for (int k = 0; k < V; ++k) res[k] = static_cast<T>(o[k]);
        const bool store = (AGAIN ? needs : live) && l.skip[i] == 0 &&
                           VBH_IN_SPAN(sy, out + l.at[i], 16);
        const int to = (gs.sub * a.cols + l.at[i]) * static_cast<int>(sizeof(T));
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, res), rsrc,
                                               store ? to : 0x7fffff00, 0, kCacheNtSc1);
        continue;
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
    if constexpr (!AHEAD) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        xr[i] = xn[i];
        gr[i] = gn[i];
      }
    }
  }
  return again;
}

// The workgroup's sums of one vector into row `row` of parts.  Lanes of a wave that hold the same
// columns are added up first.  Several groups leave theirs in the LDS, a lane's next to its
// neighbour's, and the workgroup's lanes, each with a few columns, add them in order.
template <int V, int IT>
__device__ __forceinline__ void write_sums(const NormGradArgs& a, float (&v)[IT][V], float* lds,
                                           int64_t row) {
  constexpr int F = V < 4 ? 1 : 4;  // values of an access
  typedef typename Raw<float, F>::type four;
  const int lane_tpr = a.tpr;
  const int tpr = max(lane_tpr, kWave);
  const GroupShape gs = group_shape(tpr);
  if (lane_tpr < kWave) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        for (int s = lane_tpr; s < kWave; s *= 2) v[i][k] += __shfl_xor(v[i][k], s);
      }
    }
  }
  float* out = a.parts + row * a.pitch;
  const Span sp = VBH_SPAN(a.parts, a.part_rows * a.pitch);
  // values [h F, h F + F) of vector i of lane g
  auto write = [&](int g, int i, int h, const float (&o)[F]) {
    const int first = (g + i * lane_tpr) * V, at = min(first, a.cols - V), skip = first - at;
    if (skip == 0) {
      store_any<float, F, false>(out + at + h * F, o, sp);
    } else {
#pragma unroll
      for (int k = 0; k < F; ++k)
        if (h * F + k >= skip) store_any<float, 1, false>(out + at + h * F + k, o + k, sp);
    }
  };
  if (gs.per_block == 1) {
    if (gs.g >= lane_tpr) return;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
#pragma unroll
      for (int h = 0; h < V / F; ++h) {
        float o[F];
#pragma unroll
        for (int k = 0; k < F; ++k) o[k] = v[i][h * F + k];
        write(gs.g, i, h, o);
      }
    }
    return;
  }
  four* const all = reinterpret_cast<four*>(lds);
  const int each = IT * (V / F) * tpr;  // of a group
  __syncthreads();
#pragma unroll
  for (int i = 0; i < IT; ++i) {
#pragma unroll
    for (int h = 0; h < V / F; ++h) {
      four f;
      if constexpr (F == 1) f = v[i][h];
      else f = four{v[i][4 * h], v[i][4 * h + 1], v[i][4 * h + 2], v[i][4 * h + 3]};
      all[gs.sub * each + (i * (V / F) + h) * tpr + gs.g] = f;
    }
  }
  __syncthreads();
  for (int j = static_cast<int>(threadIdx.x); j < each; j += static_cast<int>(blockDim.x)) {
    const int ih = j / tpr, g = j - ih * tpr;
    if (g >= lane_tpr) continue;
    float o[F];
#pragma unroll
    for (int k = 0; k < F; ++k) o[k] = 0.0f;
    for (int q = 0; q < gs.per_block; ++q) {
      const four f = all[q * each + j];
#pragma unroll
      for (int k = 0; k < F; ++k) {
        if constexpr (F == 1) o[k] += f;
        else o[k] += f[k];
      }
    }
    write(g, ih / (V / F), ih % (V / F), o);
  }
}

// Lanes of a workgroup at most: rows of more than two vectors for each of 1024 lanes take 512 lanes
// of twice the registers (2048 rows of 20480 bf16 values, LayerNorm: 1024 lanes of three vectors
// spill 40 registers and take 83.6 us, 512 of five 71.3).  Five vectors of whole rows just fit;
// beyond them registers spill.  16-bit LayerNorm (RMSNorm): whole rows 20 to 24 (0 to 1) registers
// at six vectors, 127 to 173 (41 to 43) at eight; ragged ones 49 to 62 (0 to 44) at five, 138 to 163
// (43 to 81) at six, 386 to 506 (228 to 349) at eight; fp32 only at eight, 12 (0) and 133 (2).
// 2048 rows, bf16, LayerNorm / RMSNorm, us (6650 GB/s would take): of 24576 values 77 / 66 (45),
// 32768 133 / 93 (61), 16385 81 / 67 (30), 20481 146 / 83 (38).
constexpr int norm_lanes(int it) { return it > 2 ? kMaxBlock / 2 : kMaxBlock; }

template <typename T, typename W, int V, int IT, bool LN, bool RAGGED, bool AHEAD>
__global__ __launch_bounds__(norm_lanes(IT)) void norm_grads(const NormGradArgs a) {
  // the row ahead; behind them all, the sums of groups other than the first
  constexpr int kBytes = norm_lanes(IT) * IT * (AHEAD ? 32 : IT > 2 ? 0 : V * 4);
  __shared__ __align__(16) char slot[kBytes > 0 ? kBytes : 16];
  __shared__ NormBuffers lds;
  NormSums<V, IT> sums;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) sums.dw[i][k] = sums.db[i][k] = 0.0f;
  }
  const bool again =
      norm_rows<T, W, V, IT, LN, RAGGED, AHEAD, false>(a, lds, slot, sums);
  if (__builtin_expect(__syncthreads_or(again), 0))
    norm_rows<T, W, V, IT, LN, RAGGED, AHEAD, true>(a, lds, slot, sums);
  if (a.parts == nullptr) return;
  float* const beside = reinterpret_cast<float*>(slot);
  write_sums<V, IT>(a, sums.dw, beside, blockIdx.x);
  if constexpr (LN) write_sums<V, IT>(a, sums.db, beside, gridDim.x + blockIdx.x);
}

// ---------------------------------------------------------------------------
// rows beyond the registers: the row's statistics first, then tiles of columns that
// read x and dy once more.  Value by value, which is what bounds them: 2048 bf16 rows of
// 40000, LayerNorm / RMSNorm, 350 / 292 us, 1024 fp32 rows of 20480 113 / 96 (bytes
// read and written once at 6650 GB/s: 74 and 38)
// ---------------------------------------------------------------------------

constexpr int kWideLanes = 256;
constexpr int kWideRows = 1 << 16;  // workgroups of a row each at a time

struct WideStat {
  float m, r, mean_g, mean_gu;
};

// One workgroup per row and every gridDim.x-th, value by value in three passes over the row (the
// second and third from the L2).
template <typename T, typename W, bool LN>
__global__ __launch_bounds__(kMaxBlock) void norm_wide_stats(const NormGradArgs a, float* stats) {
  __shared__ float mean[kMaxWaves][1], squares[kMaxWaves][1], dots[kMaxWaves][2];
  const W* w = static_cast<const W*>(a.w);
  const Span sw = VBH_SPAN(w, a.cols);
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  const int first = static_cast<int>(threadIdx.x), block = static_cast<int>(blockDim.x);
  auto at = [](const auto* p, int64_t c, const Span& sp) {
    float v;
    load_f32<std::decay_t<decltype(*p)>, 1>(p + c, &v, sp);
    return v;
  };
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.cols;
    const T* dy = static_cast<const T*>(a.dy) + row * a.cols;
    const Span sx = VBH_SPAN(x, a.cols), sg = VBH_SPAN(dy, a.cols);
    WideStat s{0.0f, 0.0f, 0.0f, 0.0f};
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

// A workgroup: 32 columns of one vector, four to a lane (whole 128-byte lines), and 64 lines of
// lanes that take up to four rows at a time, so that 256 rows take one round of loads.  Lines are
// added up through the wave, waves through the LDS, in order.  At most kPartGroups workgroups of a
// vector (a launch has fewer than 2^32 lanes), each with every kPartGroups-th 32 columns.
constexpr int kPartGroups = 1 << 16;
constexpr int kPartCols = 32;
constexpr int kPartLanes = 512;
constexpr int kPartLines = kPartLanes / (kPartCols / 4);

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
  const int line = wave * 8 + (lane >> 3);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kPartCols;
  for (int64_t col = static_cast<int64_t>(blockIdx.x) * kPartCols; col < cols; col += step) {
    const int64_t mine = col + (lane & 7) * 4;
    const float* from = parts + blockIdx.y * static_cast<int64_t>(rows) * pitch + mine;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine < pitch) {
      for (int r = line; r < rows; r += 4 * kPartLines) {
        float x[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = r + j * kPartLines;  // rows behind the last: the first of them again
          load_f32<float, 4>(from + static_cast<int64_t>(at < rows ? at : r) * pitch, x[j], sp);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] += r + j * kPartLines < rows ? x[j][i] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      for (int s = 8; s < kWave; s *= 2) v[i] += __shfl_xor(v[i], s);
    }
    if (lane < 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][lane * 4 + i] = v[i];
    }
    __syncthreads();
    const int c = static_cast<int>(threadIdx.x);
    if (c < kPartCols && col + c < cols) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kPartLanes / kWave; ++i) sum += sums[i][c];
      store_any<W, 1, false>(out + col + c, &sum, VBH_SPAN(out, cols));
    }
    if (col + step < cols) __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

constexpr int64_t kNormMaxVectors = 4 * kMaxBlock;  // of a row in registers
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
  if (nvec > kNormMaxVectors) {
    s.wide = true;
    s.grid = std::max<int64_t>(std::min<int64_t>(rows, 64), 1);
    return s;
  }
  if (nvec <= kWave) {
    s.tpr = 1;
    while (s.tpr < nvec) s.tpr *= 2;
  } else if (nvec <= 2 * kWave) {
    s.it = 2;
  } else {
    s.it = 2;
    if (nvec > 2 * kMaxBlock) {
      s.it = static_cast<int>((nvec + kMaxBlock / 2 - 1) / (kMaxBlock / 2));
      if (s.it == 7) s.it = 8;
    }
    s.tpr = static_cast<int>((nvec + int64_t(s.it) * kWave - 1) / (int64_t(s.it) * kWave)) * kWave;
  }
  // as many groups to a workgroup as leave every CU one
  s.block = std::max(s.tpr, 256 / s.tpr * s.tpr);
  while (s.block + s.tpr <= norm_lanes(s.it) && rows >= kNormCus * (s.block / s.tpr + 1)) s.block += s.tpr;
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
    const unsigned groups = static_cast<unsigned>(std::min<int64_t>(a.rows, kWideRows));
    launch_kernel(norm_wide_stats<T, W, LN>, dim3(groups), dim3(kMaxBlock), 0, stream, a, stats);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    const unsigned tiles = static_cast<unsigned>((a.cols + kWideLanes - 1) / kWideLanes);
    launch_kernel(norm_wide_apply<T, W, LN>, dim3(tiles, static_cast<unsigned>(s.grid)),
                  dim3(kWideLanes), 0, stream, a, stats);
    return hipGetLastError();
  }
  a.tpr = s.tpr;
  // nontemporal loads where the launch moves more than the last-level cache keeps from the kernel
  // before it (bf16 LayerNorm / RMSNorm, us without and with: 2048 x 8192, 100 MB, 29.5 / 23.5 and
  // 34.0 / 26.1; 8192 x 4096, 201 MB, 44.9 / 41.7 and 45.0 / 39.9)
  a.nt = 3 * a.rows * a.cols * static_cast<int64_t>(sizeof(T)) > (int64_t(128) << 20);
  constexpr int VN = Vec<T>::n;
  auto go = [&](auto kernel) {
    launch_kernel(kernel, dim3(static_cast<unsigned>(s.grid)), dim3(s.block), 0, stream, a);
    err = hipGetLastError();
  };
  const bool whole = a.cols % VN == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(a.dy) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(a.dx) % 16 == 0;
  auto by_it = [&](auto wc) {
    constexpr bool WHOLE = decltype(wc)::value;
    if (s.it == 1) go(norm_grads<T, W, VN, 1, LN, !WHOLE, false>);
    else if (s.it == 2) go(norm_grads<T, W, VN, 2, LN, !WHOLE, false>);
    else if (s.it == 5) go(norm_grads<T, W, VN, 5, LN, !WHOLE, WHOLE>);
    else if (s.it == 6) go(norm_grads<T, W, VN, 6, LN, !WHOLE, WHOLE>);
    else go(norm_grads<T, W, VN, 8, LN, !WHOLE, WHOLE>);
  };
  if (s.v == 1) go(norm_grads<T, W, 1, 1, LN, false, false>);
  else dispatch_bool(whole, by_it);
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
    const int64_t groups = (static_cast<int64_t>(a.cols) + kPartCols - 1) / kPartCols;
    launch_kernel(norm_weight_grads<W>,
                  dim3(static_cast<unsigned>(std::min<int64_t>(groups, kPartGroups)), ln ? 2 : 1),
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
