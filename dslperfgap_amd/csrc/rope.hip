// Rotation of queries and keys by position, with or without the per-head RMSNorm
// ahead of it, for gfx950.
//
//   n = x / sqrt(mean(x^2) + eps) * w,  y_a = scale * (n_a cos - n_b sin),
//   y_b = scale * (n_b cos + n_a sin)
//
// One pass: the vectors are read and written once, in 16-byte accesses, and
// everything in between is fp32, rounded once, at the store.  The angles come from
// the positions directly, so that there is no table of cosines to keep, to read or
// to outgrow.  rope.h says how vectors lie over lanes.
#include <algorithm>

#include "rope.h"

namespace vbh {

#ifndef ZPAD
#define ZPAD 5 * all(t.accesses) > 4 * all(padded)
#endif
#ifndef ZFB
#define ZFB 6
#endif
namespace {

// A wave's share: U passes over one side of token t, from head `head0` on.
template <typename T, int V, int U, bool NORM, bool ADJ, bool ANY, int MEM>
__device__ __forceinline__ void rope_share(const RopeArgs& a, const RopeSide& side,
                                           const RopeToken& t, int head0, float2* table,
                                           float* scratch) {
  const RopeLane l = rope_lane(a);
  const Span sx = VBH_SPAN(static_cast<const T*>(side.x), rope_extent(a, side.xs, side.heads));
  const RopeAngles angles(a);
  const double pos = angles.position(a, t);
  float w[V];
  if constexpr (NORM) load_weights<T, V>(a, side, l, w);
  const T* x0 = static_cast<const T*>(side.x);
  const T* from = x0 + token_offset(t, side.xs) + (head0 + l.sub) * side.xs[2] + l.at * V;
  const int64_t x_step = a.tile.per_pass * side.xs[2];
  typename Raw<T, V>::type x[U];
  bool ok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // lanes without a vector read the first values: no branch keeps the loads apart
    ok[u] = l.live && head0 + u * a.tile.per_pass + l.sub < side.heads;
    x[u] = load_any<T, V, MEM != kRopeCached>(ok[u] ? from + u * x_step : x0, sx);
  }
  angles.make(a, t, pos, table);
  wave_lds_fence();
  const RopePartner<V> partner = rope_partner<V, ANY>(a, l);
  Turn<V> turn;
  make_turn<V, ADJ, ANY>(a, l, table, turn);
  float size[U];
  if constexpr (NORM) {
    float theirs[V];
    if constexpr (!ADJ) partners<V, ANY>(w, partner, theirs);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      turn.c[i] *= w[i];
      turn.s[i] *= ADJ ? w[i ^ 1] : theirs[i];
    }
    const float inv_dim = 1.0f / static_cast<float>(a.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) size[u] = squares<T, V>(x[u]);
    vector_sums<U>(a, l, size, scratch);
#pragma unroll
    for (int u = 0; u < U; ++u) size[u] = inverse_root(fmaf(size[u], inv_dim, a.eps));
  }
  const RopeOut<T, V, MEM> out(a, side, t.t);
  const int to = (head0 + l.sub) * a.dim + l.at * V, step = a.tile.per_pass * a.dim;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    typename Raw<T, V>::type other = x[u];
    if constexpr (!ADJ) other = partners<T, V, ANY>(x[u], partner);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xi = raw_at<T, V>(x[u], i);
      const float xp = raw_at<T, V>(other, ADJ ? i ^ 1 : i);
      float y = fmaf(xi, turn.c[i], xp * turn.s[i]);
      // a value that passes takes nothing from another, which may be infinite
      if (ANY && turn.passing[i]) y = xi * turn.c[i];
      o[i] = NORM ? y * size[u] : y;
    }
    out.store(to + u * step, ok[u], o);
  }
}

// 5 waves to a SIMD: up to 96 registers, which 4 passes of 16-bit values use.
template <typename T, int V, bool NORM, bool ADJ, bool ANY, int MEM>
__global__ __launch_bounds__(kRopeBlock, ZFB) void rope_rows(const RopeArgs) {
  const RopeArgs& a = launch_args();
  extern __shared__ __align__(16) float rope_lds[];
  const int wave = wave_index();
  const uint32_t chunks = static_cast<uint32_t>(a.q.chunks + a.k.chunks);
  const uint32_t unit = blockIdx.x * static_cast<uint32_t>(kRopeWaves) + wave;
  const uint32_t turn_of = unit / chunks;
  const int64_t token = a.first + turn_of;
  if (token >= a.tokens) return;
  const int chunk = static_cast<int>(unit - turn_of * chunks);
  const RopeToken t = rope_token(a, token);
  const bool is_q = chunk < a.q.chunks;
  const RopeSide& side = a.side(!is_q);
  const int head0 =
      (is_q ? chunk : chunk - a.q.chunks) * side.per_wave * a.tile.per_pass;
  const int table_floats = rope_table_floats(a.n_freq);
  const int scratch_floats = NORM && a.tile.lanes_log2 < 0 ? kRopePasses * kRopeScratch : 0;
  float* mine = rope_lds + wave * (table_floats + scratch_floats);
  float2* table = reinterpret_cast<float2*>(mine);
  float* scratch = mine + table_floats;
  switch (side.per_wave) {
    case 1: return rope_share<T, V, 1, NORM, ADJ, ANY, MEM>(a, side, t, head0, table, scratch);
    case 2: return rope_share<T, V, 2, NORM, ADJ, ANY, MEM>(a, side, t, head0, table, scratch);
    case 3: return rope_share<T, V, 3, NORM, ADJ, ANY, MEM>(a, side, t, head0, table, scratch);
    default: return rope_share<T, V, 4, NORM, ADJ, ANY, MEM>(a, side, t, head0, table, scratch);
  }
}

// Pair by pair: one pass to a wave, a vector over up to a wave's lanes, K pairs each.
template <typename T, int K, bool NORM, bool ADJ>
__global__ __launch_bounds__(kRopeBlock) void rope_values(const RopeArgs a) {
  extern __shared__ __align__(16) float rope_lds[];
  const int wave = wave_index();
  float2* table = reinterpret_cast<float2*>(rope_lds) + wave * a.n_freq;
  const uint32_t chunks = static_cast<uint32_t>(a.q.chunks + a.k.chunks);
  const uint32_t unit = blockIdx.x * static_cast<uint32_t>(kRopeWaves) + wave;
  const uint32_t turn_of = unit / chunks;
  const int64_t token = a.first + turn_of;
  if (token >= a.tokens) return;
  const int chunk = static_cast<int>(unit - turn_of * chunks);
  const RopeToken t = rope_token(a, token);
  const RopeLane l = rope_lane(a);
  const bool is_q = chunk < a.q.chunks;
  const RopeSide& side = a.side(!is_q);
  const int head = (is_q ? chunk : chunk - a.q.chunks) * a.tile.per_pass + l.sub;
  const bool ok = l.live && head < side.heads;
  const Span sx = VBH_SPAN(static_cast<const T*>(side.x), rope_extent(a, side.xs, side.heads));
  const T* x = static_cast<const T*>(side.x) + token_offset(t, side.xs) + head * side.xs[2];
  float xa[K], xb[K], sum[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const RopePair r = rope_pair<ADJ>(a, l, k);
    xa[k] = load_value<T>(x + r.a, ok && r.has_a, sx);
    xb[k] = load_value<T>(x + r.b, ok && r.has_b, sx);
    sum[0] = fmaf(xa[k], xa[k], fmaf(xb[k], xb[k], sum[0]));
  }
  const RopeAngles angles(a);
  angles.make(a, t, angles.position(a, t), table);
  wave_lds_fence();
  float size = 1.0f;
  if constexpr (NORM) {
    vector_sums<1>(a, l, sum, nullptr);
    size = inverse_root(fmaf(sum[0], 1.0f / static_cast<float>(a.dim), a.eps));
  }
  if (!ok) return;
  const Span sy = VBH_SPAN(static_cast<T*>(side.y), a.tokens * side.heads * a.dim);
  T* y = static_cast<T*>(side.y) + (t.t * side.heads + head) * a.dim;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const RopePair r = rope_pair<ADJ>(a, l, k);
    if (!r.has_a) continue;
    float na = xa[k], nb = xb[k];
    if constexpr (NORM) {
      na *= size * load_weight<T>(a, side, r.a);
      nb *= size * (r.has_b ? load_weight<T>(a, side, r.b) : 1.0f);
    }
    float ya = na, yb = nb;
    if (r.p >= 0) {
      const float2 cs = table[r.p];
      ya = fmaf(na, cs.x, -nb * cs.y);
      yb = fmaf(nb, cs.x, na * cs.y);
    }
    store_any<T, 1>(y + r.a, &ya, sy);
    if (r.has_b) store_any<T, 1>(y + r.b, &yb, sy);
  }
}

// The passes below which a launch gives each wave one, and the workgroups of one
// launch at most.
constexpr int64_t kRopeFewPasses = 8192;
constexpr int64_t kRopeMaxGrid = ((int64_t(1) << 32) - 1) / kRopeBlock;

}  // namespace

void rope_shape(RopeArgs& a, int dt, bool adjacent, bool norm, int64_t few, int most) {
  RopeTile& t = a.tile;
  // the widest access that fits vectors and, in half accesses that are whole words,
  // the way to the partners
  t.v = dt == kF32 ? 4 : 8;
  auto fits = [&](int v) {
    const int step = dt == kF32 || v > 2 ? v / 2 : v;
    return a.dim % v == 0 && (adjacent || a.n_freq % step == 0);
  };
  while (t.v > 1 && !fits(t.v)) t.v /= 2;
  t.accesses = a.dim / t.v;
  if (t.v == 1 || t.accesses > kWave) {  // pair by pair
    t.v = 1;
    t.accesses = std::min((a.dim + 1) / 2, kWave);
    most = 1;
  }
  int padded = 1;
  while (padded < t.accesses) padded *= 2;
  auto passes = [&](const RopeSide& side, int lanes) {
    return (side.heads + kWave / lanes - 1) / (kWave / lanes);
  };
  auto all = [&](int lanes) { return passes(a.q, lanes) + passes(a.k, lanes); };
  // Vectors of no power of two of accesses: side by side without a gap, or a power of
  // two of lanes apart, which leaves lanes idle but sums in registers.  MI355X, 16384
  // tokens of 32 + 8 bf16 heads, passes and us, side by side / apart: heads of 96,
  // 9 / 10 passes, norm SIDE96 / APART96; heads of 80, 8 / 10 passes, norm SIDE80 / APART80
  t.lanes = t.v == 1 || (norm && ZPAD) ||
                    all(t.accesses) == all(padded)
                ? padded
                : t.accesses;
  t.lanes_log2 = (t.lanes & (t.lanes - 1)) == 0 ? __builtin_ctz(t.lanes) : -1;
  t.per_pass = kWave / t.lanes;
  const int pq = passes(a.q, t.lanes), pk = passes(a.k, t.lanes);
  if (a.tokens * (pq + pk) < few) most = 1;
  auto share = [&](RopeSide& side, int n) {
    // the fewest passes with a wave's own work (angles and the like) taken for two;
    // the larger share of two alike
    int best = 1 << 30;
    for (int u = 1; u <= most; ++u) {
      const int chunks = (n + u - 1) / u;
      if (chunks * (u + 2) > best) continue;
      best = chunks * (u + 2);
      side.per_wave = u;
      side.chunks = chunks;
    }
  };
  share(a.q, pq);
  share(a.k, pk);
}

hipError_t launch_rope(const RopeArgs& args, int dt, bool adjacent, bool norm, hipStream_t s) {
  RopeArgs a = args;
  rope_shape(a, dt, adjacent, norm, kRopeFewPasses, kRopePasses);
  const RopeTile& t = a.tile;
  const int chunks = a.q.chunks + a.k.chunks;
  const bool any = 2 * a.n_freq < a.dim || (!adjacent && a.n_freq % t.v != 0);
  const int64_t bytes =
      a.tokens * (a.q.heads + a.k.heads) * a.dim * (dt == kF32 ? 4 : 2);
  hipError_t err = hipErrorInvalidValue;
  auto go = [&](auto kernel, size_t floats) {
    // as many launches as keep each under 2^32 work-items
    const int64_t most = kRopeMaxGrid * kRopeWaves / chunks;  // tokens
    for (a.first = 0; a.first < a.tokens; a.first += most) {
      const int64_t units = std::min(a.tokens - a.first, most) * chunks;
      launch_kernel(kernel, dim3(static_cast<unsigned>((units + kRopeWaves - 1) / kRopeWaves)),
                    dim3(kRopeBlock), static_cast<unsigned>(floats * sizeof(float)), s, a);
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
        if (t.v == 1) {
          const size_t floats = size_t(2) * kRopeWaves * a.n_freq;
          if ((a.dim + 1) / 2 <= kWave) go(rope_values<T, 1, N, A>, floats);
          else go(rope_values<T, kRopePairs, N, A>, floats);
          return;
        }
        const size_t floats =
            size_t(kRopeWaves) * (rope_table_floats(a.n_freq) +
                                  (N && t.lanes_log2 < 0 ? kRopePasses * kRopeScratch : 0));
        auto rows = [&](auto mc) {
          constexpr int M = decltype(mc)::value;
          if (t.v == VN && !any) go(rope_rows<T, VN, N, A, false, M>, floats);
          else if (t.v == VN) go(rope_rows<T, VN, N, A, true, M>, floats);
          else if (VN == 8 && t.v == 4) go(rope_rows<T, 4, N, A, true, M>, floats);
          else go(rope_rows<T, 2, N, A, true, M>, floats);
        };
        dispatch_rope_mem(rope_mem(bytes, bytes), rows);
      });
    });
  });
  return err;
}

}  // namespace vbh
