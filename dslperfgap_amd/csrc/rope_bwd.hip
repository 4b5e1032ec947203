// Gradients of the per-head RMSNorm with the rotation behind it (rope.hip), for
// gfx950.  With u = x r, r = 1 / sqrt(mean(x^2) + eps), per vector of D values:
//
//   dn = R^T dy (the rotation back, by the same scale),  du = dn w
//   dx = r (du - u mean(du u)),  dw = sum over tokens and heads of dn u
//
// One pass over x and dy: the vector's two sums cross its lanes once, together,
// and the weights' sums stay in the lane.  A wave keeps its heads for the whole
// kernel and walks over tokens, so that a lane's 2 V sums belong to one weight;
// at the end a workgroup adds up its waves' and writes one row of sums per
// weight, and a second kernel adds the rows, all in a fixed order.
#include <algorithm>

#include "rope.h"

namespace vbh {

namespace {

template <typename T, int V, int K, int U, bool ADJ, bool PART>
__global__ __launch_bounds__(kRopeBlock) void qk_norm_rope_grads(const RopeArgs a, float* parts) {
  extern __shared__ float2 rope_tables[];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int chunk = static_cast<int>(blockIdx.x % static_cast<uint32_t>(a.chunks));
  const int walker = static_cast<int>(blockIdx.x / static_cast<uint32_t>(a.chunks));
  const int walkers = static_cast<int>(gridDim.x / static_cast<uint32_t>(a.chunks));
  const RopeLane l = rope_lane(a, chunk);
  float2* table = rope_tables + wave * U * a.slots;

  const int hh = l.is_q ? l.head : l.head - a.q.heads;
  const T* x = static_cast<const T*>(l.is_q ? a.q.x : a.k.x) +
               hh * (l.is_q ? a.q.xs[2] : a.k.xs[2]);
  const T* g = static_cast<const T*>(l.is_q ? a.q.g : a.k.g) +
               hh * (l.is_q ? a.q.gs[2] : a.k.gs[2]);
  T* y = static_cast<T*>(l.is_q ? a.q.y : a.k.y) + static_cast<int64_t>(hh) * a.dim;
  const Span sx = pick_span(
      l.is_q, VBH_SPAN(static_cast<const T*>(a.q.x), rope_extent(a, a.q.xs, a.q.heads)),
      VBH_SPAN(static_cast<const T*>(a.k.x), rope_extent(a, a.k.xs, a.k.heads)));
  const Span sg = pick_span(
      l.is_q, VBH_SPAN(static_cast<const T*>(a.q.g), rope_extent(a, a.q.gs, a.q.heads)),
      VBH_SPAN(static_cast<const T*>(a.k.g), rope_extent(a, a.k.gs, a.k.heads)));
  const Span sy =
      pick_span(l.is_q, VBH_SPAN(static_cast<T*>(a.q.y), a.tokens * a.q.heads * a.dim),
                VBH_SPAN(static_cast<T*>(a.k.y), a.tokens * a.k.heads * a.dim));

  RopePiece p[K];
  float w[K][2 * V], dw[K][2 * V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    p[k] = rope_piece<V, ADJ>(a, l, k);
    load_weights<T, V>(a, l, p[k], w[k]);
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) dw[k][i] = 0.0f;
  }
  const float inv_dim = 1.0f / static_cast<float>(a.dim);

  const int64_t step = static_cast<int64_t>(walkers) * kRopeWaves * U;
  for (int64_t t0 = (static_cast<int64_t>(walker) * kRopeWaves + wave) * U; t0 < a.tokens;
       t0 += step) {
    const int b0 = a.batch > 1 ? static_cast<int>(static_cast<uint32_t>(t0) /
                                                  static_cast<uint32_t>(a.seq)) : 0;
    const int s0 = static_cast<int>(t0 - static_cast<int64_t>(b0) * a.seq);
    typename Raw<T, V>::type xa[U][K], xb[U][K], ga[U][K], gb[U][K];
    int b = b0, s = s0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = t0 + u < a.tokens;
      const int64_t xq = b * a.q.xs[0] + s * a.q.xs[1], xk = b * a.k.xs[0] + s * a.k.xs[1];
      const int64_t gq = b * a.q.gs[0] + s * a.q.gs[1], gk = b * a.k.gs[0] + s * a.k.gs[1];
      const T* xt = x + (l.is_q ? xq : xk);
      const T* gt = g + (l.is_q ? gq : gk);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const typename Raw<T, V>::type zero{};
        xa[u][k] = there && p[k].has_a ? load_any<T, V>(xt + p[k].a, sx) : zero;
        xb[u][k] = there && p[k].has_b ? load_any<T, V>(xt + p[k].b, sx) : zero;
        ga[u][k] = there && p[k].has_a ? load_any<T, V>(gt + p[k].a, sg) : zero;
        gb[u][k] = there && p[k].has_b ? load_any<T, V>(gt + p[k].b, sg) : zero;
      }
      if (++s == a.seq) {
        s = 0;
        ++b;
      }
    }
    wave_lds_fence();
    make_angles<U>(a, t0, b0, s0, table);
    wave_lds_fence();

#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u >= a.tokens) break;
      float dn[K][2 * V];
      float sums[2] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float c[V], si[V];
        if (p[k].has_a) {
          piece_angles<V, ADJ>(a, p[k], table + u * a.slots, c, si);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) c[i] = si[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          int i0, i1;
          pair_at<V, ADJ>(i, i0, i1);
          const float g0 = i0 < V ? raw_at<T, V>(ga[u][k], i0) : raw_at<T, V>(gb[u][k], i0 - V);
          const float g1 = i1 < V ? raw_at<T, V>(ga[u][k], i1) : raw_at<T, V>(gb[u][k], i1 - V);
          const float x0 = i0 < V ? raw_at<T, V>(xa[u][k], i0) : raw_at<T, V>(xb[u][k], i0 - V);
          const float x1 = i1 < V ? raw_at<T, V>(xa[u][k], i1) : raw_at<T, V>(xb[u][k], i1 - V);
          // sin_scale is that of the rotation back
          float n0 = fmaf(g0, c[i], -g1 * si[i]), n1 = fmaf(g1, c[i], g0 * si[i]);
          if (PART && rope_pair<V, ADJ>(a, p[k], i) >= a.n_freq) {
            n0 = g0;
            n1 = g1;
          }
          dn[k][i0] = n0;
          dn[k][i1] = n1;
          sums[0] = fmaf(x0, x0, fmaf(x1, x1, sums[0]));
          sums[1] = fmaf(n0 * w[k][i0], x0, fmaf(n1 * w[k][i1], x1, sums[1]));
        }
      }
      group_sums<2>(sums, a.group_log2);
      const float r = inverse_root(fmaf(sums[0], inv_dim, a.eps));
      const float mean = sums[1] * r * inv_dim;
      const int64_t row = (t0 + u) * (l.is_q ? a.q.heads : a.k.heads) * a.dim;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float o[2 * V];
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) {
          const float v = i < V ? raw_at<T, V>(xa[u][k], i) : raw_at<T, V>(xb[u][k], i - V);
          const float unit = v * r;
          dw[k][i] = fmaf(dn[k][i], unit, dw[k][i]);
          o[i] = r * fmaf(dn[k][i], w[k][i], -unit * mean);
        }
        if (p[k].has_a) store_any<T, V>(y + row + p[k].a, o, sy);
        if (p[k].has_b) store_any<T, V>(y + row + p[k].b, o + V, sy);
      }
    }
  }
  if (parts == nullptr) return;

  // the workgroup's sums: every vector's place in the LDS, then one lane per value
  const int per_wave = kWave >> a.group_log2;
  float* sums = reinterpret_cast<float*>(rope_tables);
  __syncthreads();
  const int mine = (wave * per_wave + (static_cast<int>(threadIdx.x) & (kWave - 1)) /
                                          (1 << a.group_log2)) * a.dim;
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (p[k].has_a) sums[mine + p[k].a + i] = dw[k][i];
      if (p[k].has_b) sums[mine + p[k].b + i] = dw[k][V + i];
    }
  }
  __syncthreads();
  // rows of sums: q's chunks of every walker, then k's
  const RopeRows rows = rope_rows_of(a.q.heads, a.k.heads, per_wave);
  const Span sp = VBH_SPAN(parts, static_cast<int64_t>(walkers) * (rows.q + rows.k) * a.dim);
  const int from = chunk * per_wave;
  const int cut = min(max(a.q.heads - from, 0), per_wave);                // first k vector
  const int end = min(max(a.q.heads + a.k.heads - from, 0), per_wave);
  for (int d = static_cast<int>(threadIdx.x); d < a.dim; d += kRopeBlock) {
    float q = 0.0f, kk = 0.0f;
    for (int v = 0; v < kRopeWaves; ++v) {
      for (int h = 0; h < cut; ++h) q += sums[(v * per_wave + h) * a.dim + d];
      for (int h = cut; h < end; ++h) kk += sums[(v * per_wave + h) * a.dim + d];
    }
    if (cut > 0) {
      float* to = parts + (static_cast<int64_t>(walker) * rows.q + chunk) * a.dim + d;
      store_any<float, 1, false>(to, &q, sp);
    }
    if (end > cut) {
      float* to = parts + (static_cast<int64_t>(walkers) * rows.q +
                           static_cast<int64_t>(walker) * rows.k + chunk - rows.k_from) * a.dim + d;
      store_any<float, 1, false>(to, &kk, sp);
    }
  }
}

// Sums over the rows of parts: workgroup (tile, side), 16 columns, 64 lines of lanes.
constexpr int kSumCols = 16;
constexpr int kSumLines = 64;

template <typename W>
__global__ __launch_bounds__(kSumCols * kSumLines) void qk_weight_grads(
    const float* parts, int64_t q_rows, int64_t k_rows, int dim, W* dq, W* dk) {
  __shared__ float lines[kSumLines][kSumCols + 1];
  const bool is_q = blockIdx.y == 0;
  W* out = is_q ? dq : dk;
  if (out == nullptr) return;
  const Span sp = VBH_SPAN(parts, (q_rows + k_rows) * dim);
  const Span so = VBH_SPAN(out, dim);
  const int64_t first = is_q ? 0 : q_rows, rows = is_q ? q_rows : k_rows;
  const int c = static_cast<int>(threadIdx.x) % kSumCols;
  const int line = static_cast<int>(threadIdx.x) / kSumCols;
  const int d = static_cast<int>(blockIdx.x) * kSumCols + c;
  float sum = 0.0f;
  if (d < dim) {
#pragma unroll 8
    for (int64_t r = line; r < rows; r += kSumLines)
      sum += load_any<float, 1, false>(parts + (first + r) * dim + d, sp);
  }
  lines[line][c] = sum;
  __syncthreads();
  if (line != 0 || d >= dim) return;
  for (int i = 1; i < kSumLines; ++i) sum += lines[i][c];
  store_any<W, 1, false>(out + d, &sum, so);
}

// Tokens that a wave takes at a time, and the workgroups of a launch: as many as
// the card holds at once.
constexpr int kGradTokens = 2;
constexpr int64_t kGradBlocks = 1024;

struct GradShape {
  RopeShape sh;
  int u;
  int64_t walkers;
};

GradShape grad_shape(const RopeArgs& a, int dt, bool adjacent) {
  GradShape g;
  g.sh = rope_shape(a, dt, adjacent);
  const bool wide = g.sh.k == 1 && g.sh.v == (dt == kF32 ? 4 : 8);
  g.u = wide && a.tokens * g.sh.chunks >= kRopeFewWaves ? kGradTokens : 1;
  const int64_t tiles = (a.tokens + kRopeWaves * g.u - 1) / (kRopeWaves * g.u);
  const int64_t most = std::max<int64_t>(kGradBlocks / std::max(g.sh.chunks, 1), 1);
  const int64_t turns = (tiles + most - 1) / most;  // of the busiest walker
  // none of an empty launch: the weights' gradients are then sums of no rows
  g.walkers = turns > 0 && g.sh.chunks > 0 ? (tiles + turns - 1) / turns : 0;
  return g;
}

}  // namespace

int64_t rope_bwd_part_floats(const RopeArgs& a, int dt, bool adjacent) {
  const GradShape g = grad_shape(a, dt, adjacent);
  const RopeRows rows = rope_rows_of(a.q.heads, a.k.heads, kWave >> g.sh.group_log2);
  return g.walkers * (rows.q + rows.k) * a.dim;
}

hipError_t launch_qk_norm_rope_bwd(const RopeArgs& args, int dt, bool adjacent, void* dq_weight,
                                   void* dk_weight, float* parts, hipStream_t s) {
  const GradShape gs = grad_shape(args, dt, adjacent);
  const RopeShape& sh = gs.sh;
  RopeArgs a = args;
  a.group_log2 = sh.group_log2;
  a.slot_log2 = sh.slot_log2;
  a.chunks = sh.chunks;
  const bool part = 2 * a.n_freq < a.dim;
  const bool sums = dq_weight != nullptr || dk_weight != nullptr;
  const int per_wave = kWave >> sh.group_log2;
  hipError_t err = hipSuccess;
  if (gs.walkers * a.chunks > 0) {
    const size_t lds = std::max(kRopeWaves * gs.u * a.slots * sizeof(float2),
                                sums ? kRopeWaves * per_wave * a.dim * sizeof(float) : 0);
    auto go = [&](auto kernel) {
      launch_kernel(kernel, dim3(static_cast<unsigned>(gs.walkers * a.chunks)), dim3(kRopeBlock),
                    static_cast<unsigned>(lds), s, a, sums ? parts : nullptr);
      err = hipGetLastError();
    };
    dispatch_float_type(dt, [&](auto tt) {
      using T = typename decltype(tt)::type;
      constexpr int VN = Vec<T>::n;
      dispatch_bool(adjacent, [&](auto ac) {
        constexpr bool A = decltype(ac)::value;
        if (sh.k > 1) return go(qk_norm_rope_grads<T, 1, kRopeMaxK, 1, A, true>);
        if (sh.v == VN)
          return dispatch_bool(part, [&](auto pc) {
            constexpr bool P = decltype(pc)::value;
            if (gs.u == 1) go(qk_norm_rope_grads<T, VN, 1, 1, A, P>);
            else go(qk_norm_rope_grads<T, VN, 1, kGradTokens, A, P>);
          });
        if constexpr (VN == 8)
          if (sh.v == 4) return go(qk_norm_rope_grads<T, 4, 1, 1, A, true>);
        if (sh.v == 2) return go(qk_norm_rope_grads<T, 2, 1, 1, A, true>);
        go(qk_norm_rope_grads<T, 1, 1, 1, A, true>);
      });
    });
  }
  if (err != hipSuccess || !sums) return err;
  const RopeRows rows = rope_rows_of(a.q.heads, a.k.heads, per_wave);
  auto sum = [&](auto tag) {
    using W = typename decltype(tag)::type;
    launch_kernel(qk_weight_grads<W>, dim3((a.dim + kSumCols - 1) / kSumCols, 2),
                  dim3(kSumCols * kSumLines), 0, s, parts, gs.walkers * rows.q,
                  gs.walkers * rows.k, a.dim, static_cast<W*>(dq_weight),
                  static_cast<W*>(dk_weight));
    err = hipGetLastError();
  };
  if (a.w_f32) sum(TypeTag<float>{});
  else dispatch_float_type(dt, sum);
  return err;
}

}  // namespace vbh
