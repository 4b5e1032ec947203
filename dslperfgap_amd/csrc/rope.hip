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

namespace {

// A wave's share: U passes over one side of token t, from head `head0` on.
template <typename T, int V, int U, bool NORM, bool ADJ, int WAY, int MEM>
__device__ __forceinline__ void rope_share(const RopeArgs& a, const RopeSide& side,
                                           const RopeToken& t, int head0, float* lds) {
  const RopeLane l = rope_lane(a);
  const Span sx = VBH_SPAN(static_cast<const T*>(side.x), rope_extent(a, side.xs, side.heads));
  const RopeLds parts = rope_lds_of(a, NORM ? kRopePasses : 0, kRopePasses);
  float2* table = reinterpret_cast<float2*>(lds);
  float* scratch = lds + parts.table;
  char* rows = reinterpret_cast<char*>(scratch + parts.scratch);
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
  const RopePartners<T, V, U, WAY> partners(a, l, x, rows);
  Turn<V> turn;
  make_turn<V, ADJ, WAY>(a, l, table, turn);
  float size[U];
  if constexpr (NORM) {
    float theirs[V];
    if constexpr (!ADJ) partner_weights<T, V, WAY>(a, side, l, partners.p, w, theirs);
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
    float other[V], o[V];
    if constexpr (!ADJ) partners.get(x[u], u, other);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float xi = raw_at<T, V>(x[u], i);
      float xp = ADJ ? raw_at<T, V>(x[u], i ^ 1) : other[i];
      if constexpr (NORM) {  // first: a product with C or S may pass the range of 32 bits
        xi *= size[u];
        xp *= size[u];
      }
      const float y = fmaf(xi, turn.c[i], xp * turn.s[i]);
      // a value that passes takes nothing from another, which may be infinite
      o[i] = WAY != kRopeWhole && turn.passing[i] ? xi * turn.c[i] : y;
    }
    out.store(to + u * step, ok[u], o);
  }
}

// 6 waves to a SIMD, 80 registers.  MI355X, norm and rotation of 16384 tokens of 40 bf16
// heads, us at 5 / 6 / 7 / 8 waves, in turn: heads of 128, half pairing 53.7 / 54.0 / 54.6 /
// 69.2 (registers spill at 8), adjacent 54.6 / 51.5 / 51.5 / 50.9; of 96 49.8 / 49.9 / 49.6 /
// 62.7 and 50.9 / 44.7 / 44.7 / 42.9.  Without the norm all four take the same within 1%.
template <typename T, int V, bool NORM, bool ADJ, int WAY, int MEM>
__global__ __launch_bounds__(kRopeBlock, 6) void rope_rows(const RopeArgs) {
  const RopeArgs& a = launch_args();
  extern __shared__ __align__(16) float rope_lds[];
  const int wave = wave_index();
  float* lds = rope_lds + wave * rope_lds_of(a, NORM ? kRopePasses : 0, kRopePasses).all();
  const uint32_t chunks = static_cast<uint32_t>(a.q().chunks + a.k().chunks);
  const uint32_t unit = blockIdx.x * static_cast<uint32_t>(kRopeWaves) + wave;
  const uint32_t turn_of = unit / chunks;
  const int64_t token = a.first + turn_of;
  if (token >= a.tokens) return;
  const int chunk = static_cast<int>(unit - turn_of * chunks);
  const RopeToken t = rope_token(a, token);
  const bool is_k = chunk >= a.q().chunks;
  const RopeSide& side = a.side(is_k);
  const int head0 = (is_k ? chunk - a.q().chunks : chunk) * side.per_wave * a.tile.per_pass;
  switch (side.per_wave) {
    case 1: return rope_share<T, V, 1, NORM, ADJ, WAY, MEM>(a, side, t, head0, lds);
    case 2: return rope_share<T, V, 2, NORM, ADJ, WAY, MEM>(a, side, t, head0, lds);
    case 3: return rope_share<T, V, 3, NORM, ADJ, WAY, MEM>(a, side, t, head0, lds);
    default: return rope_share<T, V, 4, NORM, ADJ, WAY, MEM>(a, side, t, head0, lds);
  }
}

// Pair by pair: one pass to a wave, a vector over up to a wave's lanes, K pairs each.
template <typename T, int K, bool NORM, bool ADJ>
__global__ __launch_bounds__(kRopeBlock) void rope_values(const RopeArgs a) {
  extern __shared__ __align__(16) float rope_lds[];
  const int wave = wave_index();
  float2* table =
      reinterpret_cast<float2*>(rope_lds + wave * rope_lds_of(a, 0, 0).table);
  const uint32_t chunks = static_cast<uint32_t>(a.q().chunks + a.k().chunks);
  const uint32_t unit = blockIdx.x * static_cast<uint32_t>(kRopeWaves) + wave;
  const uint32_t turn_of = unit / chunks;
  const int64_t token = a.first + turn_of;
  if (token >= a.tokens) return;
  const int chunk = static_cast<int>(unit - turn_of * chunks);
  const RopeToken t = rope_token(a, token);
  const RopeLane l = rope_lane(a);
  const bool is_q = chunk < a.q().chunks;
  const RopeSide& side = a.side(!is_q);
  const int head = (is_q ? chunk : chunk - a.q().chunks) * a.tile.per_pass + l.sub;
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
      // the vector first: size * weight may leave the range of 32 bits
      na = na * size * load_weight<T>(a, side, r.a);
      nb = nb * size * (r.has_b ? load_weight<T>(a, side, r.b) : 1.0f);
    }
    float ya = na, yb = nb;
    if (r.p >= 0) {
      const float2 cs = table[table_place(r.p)];
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

void rope_shape(RopeArgs& a, int dt, bool adjacent, bool norm, int64_t many, int least,
                int most, bool even) {
  RopeTile& t = a.tile;
  const int elt = dt == kF32 ? 4 : 2;
  t.v = 16 / elt;  // the widest access that vectors are a whole number of
  while (t.v > 1 && a.dim % t.v != 0) t.v /= 2;
  t.accesses = a.dim / t.v;
  if (t.v == 1 || t.accesses > kWave) {  // pair by pair
    t.v = 1;
    t.accesses = std::min((a.dim + 1) / 2, kWave);
    least = most = 1;
  }
  // half accesses that are whole words find their partners in one lane each
  a.gather = !adjacent && t.v > 1 && a.n_freq % (dt == kF32 || t.v > 2 ? t.v / 2 : t.v) != 0;
  int padded = 1;
  while (padded < t.accesses) padded *= 2;
  auto passes = [&](const RopeSide& side, int lanes) {
    return (side.heads + kWave / lanes - 1) / (kWave / lanes);
  };
  auto all = [&](int lanes) { return passes(a.q(), lanes) + passes(a.k(), lanes); };
  // Vectors of no power of two of accesses: side by side without a gap, or a power of
  // two of lanes apart, which leaves lanes idle but sums in registers.  MI355X, 16384
  // tokens of 32 + 8 bf16 heads, us side by side / apart: heads of 96 (9 / 10 passes)
  // forward 53.4 / 49.5, backward 87.0 / 77.6; heads of 80 (8 / 10 passes) 52.2 / 51.7 and
  // 70.3 / 74.5; heads of 72 (7 / 10) 55.1 / 55.0 and 75.2 / 80.1
  t.lanes = t.v == 1 || (norm && 5 * all(t.accesses) > 4 * all(padded)) ||
                    all(t.accesses) == all(padded)
                ? padded
                : t.accesses;
  t.lanes_log2 = (t.lanes & (t.lanes - 1)) == 0 ? __builtin_ctz(t.lanes) : -1;
  t.per_pass = kWave / t.lanes;
  const int pq = passes(a.q(), t.lanes), pk = passes(a.k(), t.lanes);
  const int64_t total = a.tokens * (pq + pk);
  if (a.n_freq <= kWave && t.lanes_log2 >= 0 && t.lanes == t.accesses && t.v * elt == 16)
    most = std::min(most, 4);
  most = total < many
             ? 1
             : static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(total / many, least)));
  auto share = [&](RopeSide& side, int n) {
    // the fewest passes with a wave's own work (angles and the like) taken for two; the
    // larger share of two alike
    int best = 1 << 30;
    for (int u = 1; u <= most; u += even && u > 1 ? 2 : 1) {
      const int chunks = (n + u - 1) / u;
      if (chunks * (u + 2) > best) continue;
      best = chunks * (u + 2);
      side.per_wave = u;
      side.chunks = chunks;
    }
  };
  share(a.q(), pq);
  share(a.k(), pk);
}

hipError_t launch_rope(const RopeArgs& args, int dt, bool adjacent, bool norm, hipStream_t s) {
  RopeArgs a = args;
  rope_shape(a, dt, adjacent, norm, kRopeFewPasses, kRopePasses, kRopePasses, false);
  const RopeTile& t = a.tile;
  const int chunks = a.q().chunks + a.k().chunks;
  const bool whole = 2 * a.n_freq == a.dim && (adjacent || a.n_freq % t.v == 0);
  const int64_t bytes =
      a.tokens * (a.q().heads + a.k().heads) * a.dim * (dt == kF32 ? 4 : 2);
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
          const size_t floats = size_t(kRopeWaves) * rope_lds_of(a, 0, 0).table;
          if ((a.dim + 1) / 2 <= kWave) go(rope_values<T, 1, N, A>, floats);
          else go(rope_values<T, kRopePairs, N, A>, floats);
          return;
        }
        const size_t floats =
            size_t(kRopeWaves) * rope_lds_of(a, N ? kRopePasses : 0, kRopePasses).all();
        auto rows = [&](auto mc) {
          constexpr int M = decltype(mc)::value;
          if (t.v == VN && whole) return go(rope_rows<T, VN, N, A, kRopeWhole, M>, floats);
          dispatch_bool(a.gather != 0, [&](auto gc) {
            constexpr int W = decltype(gc)::value && !A ? kRopeGather : kRopeHalves;
            if (t.v == VN) go(rope_rows<T, VN, N, A, W, M>, floats);
            else if (VN == 8 && t.v == 4) go(rope_rows<T, 4, N, A, W, M>, floats);
            else go(rope_rows<T, 2, N, A, W, M>, floats);
          });
        };
        dispatch_rope_mem(rope_mem(bytes, bytes), rows);
      });
    });
  });
  return err;
}

}  // namespace vbh
