// Rotation of queries and keys by position, with or without the per-head RMSNorm
// ahead of it, for gfx950.
//
//   n = x / sqrt(mean(x^2) + eps) * w,  y_a = scale * (n_a cos - n_b sin),
//   y_b = scale * (n_b cos + n_a sin)
//
// One pass: a lane holds both members of its pairs (rope.h), so that the rotation
// crosses no lanes and the norm costs one sum over the vector's lanes.  The
// vectors are read and written once, in 16-byte pieces; everything in between is
// fp32 and rounded once, at the store.  The angles come from the positions
// directly, one sincos per lane for a token's whole wave, through the LDS, so that
// there is no table of cosines to keep, to read or to outgrow.
#include <algorithm>

#include "rope.h"

namespace vbh {

namespace {

template <typename T, int V, int K, int U, bool NORM, bool ADJ, bool PART>
__global__ __launch_bounds__(kRopeBlock) void rope_rows(const RopeArgs a) {
  extern __shared__ float2 rope_tables[];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const uint32_t tile = blockIdx.x / static_cast<uint32_t>(a.chunks);
  const int chunk = static_cast<int>(blockIdx.x - tile * static_cast<uint32_t>(a.chunks));
  const int64_t t0 = a.first + (static_cast<int64_t>(tile) * kRopeWaves + wave) * U;
  if (t0 >= a.tokens) return;
  const RopeLane l = rope_lane(a, chunk);
  float2* table = rope_tables + wave * U * a.slots;
  const int b0 = a.batch > 1 ? static_cast<int>(static_cast<uint32_t>(t0) /
                                                static_cast<uint32_t>(a.seq)) : 0;
  const int s0 = static_cast<int>(t0 - static_cast<int64_t>(b0) * a.seq);

  const int hh = l.is_q ? l.head : l.head - a.q.heads;
  const T* x = static_cast<const T*>(l.is_q ? a.q.x : a.k.x) +
               hh * (l.is_q ? a.q.xs[2] : a.k.xs[2]);
  T* y = static_cast<T*>(l.is_q ? a.q.y : a.k.y) + static_cast<int64_t>(hh) * a.dim;
  const Span sx = pick_span(
      l.is_q, VBH_SPAN(static_cast<const T*>(a.q.x), rope_extent(a, a.q.xs, a.q.heads)),
      VBH_SPAN(static_cast<const T*>(a.k.x), rope_extent(a, a.k.xs, a.k.heads)));
  const Span sy =
      pick_span(l.is_q, VBH_SPAN(static_cast<T*>(a.q.y), a.tokens * a.q.heads * a.dim),
                VBH_SPAN(static_cast<T*>(a.k.y), a.tokens * a.k.heads * a.dim));

  RopePiece p[K];
#pragma unroll
  for (int k = 0; k < K; ++k) p[k] = rope_piece<V, ADJ>(a, l, k);

  typename Raw<T, V>::type ra[U][K], rb[U][K];
  int b = b0, s = s0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool there = t0 + u < a.tokens;
    const int64_t off_q = b * a.q.xs[0] + s * a.q.xs[1];
    const int64_t off_k = b * a.k.xs[0] + s * a.k.xs[1];
    const T* xt = x + (l.is_q ? off_q : off_k);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      ra[u][k] = there && p[k].has_a ? load_any<T, V>(xt + p[k].a, sx) : typename Raw<T, V>::type{};
      rb[u][k] = there && p[k].has_b ? load_any<T, V>(xt + p[k].b, sx) : typename Raw<T, V>::type{};
    }
    if (++s == a.seq) {
      s = 0;
      ++b;
    }
  }
  float w[NORM ? K : 1][2 * V];
  if constexpr (NORM) {
#pragma unroll
    for (int k = 0; k < K; ++k) load_weights<T, V>(a, l, p[k], w[k]);
  }
  make_angles<U>(a, t0, b0, s0, table);
  wave_lds_fence();

  float size[U];
  if constexpr (NORM) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float va = raw_at<T, V>(ra[u][k], i), vb = raw_at<T, V>(rb[u][k], i);
          sum = fmaf(va, va, sum);
          sum = fmaf(vb, vb, sum);
        }
      }
      size[u] = sum;
    }
    group_sums<U>(size, a.group_log2);
    const float inv_dim = 1.0f / static_cast<float>(a.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) size[u] = inverse_root(fmaf(size[u], inv_dim, a.eps));
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (t0 + u >= a.tokens) break;
    T* yt = y + (t0 + u) * (l.is_q ? a.q.heads : a.k.heads) * a.dim;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!p[k].has_a) continue;
      float c[V], si[V], o[2 * V];
      piece_angles<V, ADJ>(a, p[k], table + u * a.slots, c, si);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        int i0, i1;
        pair_at<V, ADJ>(i, i0, i1);
        float x0 = i0 < V ? raw_at<T, V>(ra[u][k], i0) : raw_at<T, V>(rb[u][k], i0 - V);
        float x1 = i1 < V ? raw_at<T, V>(ra[u][k], i1) : raw_at<T, V>(rb[u][k], i1 - V);
        if constexpr (NORM) {
          x0 *= w[k][i0];
          x1 *= w[k][i1];
          c[i] *= size[u];
          si[i] *= size[u];
        }
        o[i0] = fmaf(x0, c[i], -x1 * si[i]);
        o[i1] = fmaf(x1, c[i], x0 * si[i]);
        // a value that passes takes nothing from its partner, which may be infinite
        if (PART && rope_pair<V, ADJ>(a, p[k], i) >= a.n_freq) {
          o[i0] = x0 * c[i];
          o[i1] = x1 * c[i];
        }
      }
      store_any<T, V>(yt + p[k].a, o, sy);
      if (p[k].has_b) store_any<T, V>(yt + p[k].b, o + V, sy);
    }
  }
}

// Tokens that a wave takes, and the workgroups of one launch at most.
constexpr int kRopeTokens = 4;
constexpr int64_t kRopeMaxGrid = ((int64_t(1) << 32) - 1) / kRopeBlock;

}  // namespace

RopeShape rope_shape(const RopeArgs& a, int dt, bool adjacent) {
  // the widest piece that the pairs and the passing values fill whole
  RopeShape sh;
  sh.v = dt == kF32 ? 4 : 8;
  auto fits = [&](int v) {
    if (v == 1) return true;
    if (a.dim % (2 * v) != 0) return false;
    return adjacent || a.n_freq % v == 0;
  };
  while (!fits(sh.v)) sh.v /= 2;
  int lanes = (a.slots + sh.v - 1) / sh.v;
  if (lanes > kWave) {  // long vectors of odd sizes: a wave walks them value by value
    sh.v = 1;
    sh.k = kRopeMaxK;
    lanes = kWave;
  }
  while ((1 << sh.group_log2) < lanes) ++sh.group_log2;
  while ((1 << sh.slot_log2) < a.slots && (1 << sh.slot_log2) < kWave) ++sh.slot_log2;
  const int per_wave = kWave >> sh.group_log2;
  sh.chunks = (a.q.heads + a.k.heads + per_wave - 1) / per_wave;
  return sh;
}

hipError_t launch_rope(const RopeArgs& args, int dt, bool adjacent, bool norm, hipStream_t s) {
  const RopeShape sh = rope_shape(args, dt, adjacent);
  RopeArgs a = args;
  a.group_log2 = sh.group_log2;
  a.slot_log2 = sh.slot_log2;
  a.chunks = sh.chunks;
  const bool part = 2 * a.n_freq < a.dim;
  const bool few = a.tokens * a.chunks < kRopeFewWaves;
  hipError_t err = hipErrorInvalidValue;
  auto go = [&](auto kernel, int u) {
    const unsigned lds = static_cast<unsigned>(kRopeWaves * u * a.slots * sizeof(float2));
    // as many launches as keep each under 2^32 work-items
    const int64_t per_tile = kRopeWaves * u;
    const int64_t most = kRopeMaxGrid / a.chunks;
    for (a.first = 0; a.first < a.tokens; a.first += most * per_tile) {
      const int64_t tiles = std::min((a.tokens - a.first + per_tile - 1) / per_tile, most);
      launch_kernel(kernel, dim3(static_cast<unsigned>(tiles * a.chunks)), dim3(kRopeBlock), lds,
                    s, a);
      err = hipGetLastError();
      if (err != hipSuccess) return;
    }
  };
  dispatch_float_type(dt, [&](auto tt) {
    using T = typename decltype(tt)::type;
    constexpr int VN = Vec<T>::n;
    dispatch_bool(norm, [&](auto nc) {
      constexpr bool N = decltype(nc)::value;
      dispatch_bool(adjacent, [&](auto ac) {
        constexpr bool A = decltype(ac)::value;
        if (sh.k > 1) return go(rope_rows<T, 1, kRopeMaxK, 1, N, A, true>, 1);
        if (sh.v == VN)
          return dispatch_bool(part, [&](auto pc) {
            constexpr bool P = decltype(pc)::value;
            if (few) go(rope_rows<T, VN, 1, 1, N, A, P>, 1);
            else go(rope_rows<T, VN, 1, kRopeTokens, N, A, P>, kRopeTokens);
          });
        if constexpr (VN == 8)
          if (sh.v == 4) return go(rope_rows<T, 4, 1, 1, N, A, true>, 1);
        if (sh.v == 2) return go(rope_rows<T, 2, 1, 1, N, A, true>, 1);
        go(rope_rows<T, 1, 1, 1, N, A, true>, 1);
      });
    });
  });
  return err;
}

}  // namespace vbh
