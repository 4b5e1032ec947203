// Gradients of the per-head RMSNorm with the rotation behind it (rope.hip), for
// gfx950.  With u = x r, r = 1 / sqrt(mean(x^2) + eps), per vector of D values:
//
//   dn = R^T dy (the rotation back, by the same scale),  du = dn w
//   dx = r (du - u mean(du u)),  dw = sum over tokens and heads of dn u
//
// One pass over x and dy, the vectors over lanes as in the forward; only dy has
// partners.  The weights' sums stay in the lane: a wave walks over tokens and
// keeps V sums for the queries' weight and V for the keys'.  At the end a workgroup
// adds up its waves' and writes one row of sums per weight, and a second kernel
// adds the rows, all in a fixed order.
#include <algorithm>

#include "rope.h"

namespace vbh {

namespace {

constexpr int kGradPasses = 2;  // that a wave has in registers at a time

// Workgroups that have queries' waves and that have keys' (one may have both), and
// the first of the latter.
struct RopeRows {
  int q, k, k_from;
};
__host__ __device__ inline RopeRows rope_rows_of(const RopeArgs& a) {
  const int q = a.q().chunks * a.q().walkers, k = a.k().chunks * a.k().walkers;
  RopeRows r;
  r.q = (q + kRopeWaves - 1) / kRopeWaves;
  r.k_from = q / kRopeWaves;
  r.k = k > 0 ? (q + k + kRopeWaves - 1) / kRopeWaves - r.k_from : 0;
  return r;
}

// A wave's part of the launch: share `chunk` of one side's passes, of every
// walkers-th token from `token` on.  Queries' waves come first; none behind them all.
struct RopeWalk {
  bool is_q, live;
  int chunk, token;
};
__device__ __forceinline__ RopeWalk rope_walk(const RopeArgs& a, int wave) {
  const int w = static_cast<int>(blockIdx.x) * kRopeWaves + wave;
  const int q = a.q().chunks * a.q().walkers, k = a.k().chunks * a.k().walkers;
  const bool is_q = w < q;
  const uint32_t i = static_cast<uint32_t>(is_q ? w : w - q);
  const uint32_t chunks = static_cast<uint32_t>(max(is_q ? a.q().chunks : a.k().chunks, 1));
  const uint32_t token = i / chunks;
  return RopeWalk{is_q, w < q + k, static_cast<int>(i - token * chunks),
                  static_cast<int>(token)};
}

// The workgroup's row of sums for each weight that its waves have worked on: `sums`
// holds `each` vectors of every wave's.  parts: q's rows, then k's.
__device__ __forceinline__ void write_part(const RopeArgs& a, const float* sums, int each,
                                           float* parts) {
  const RopeRows rows = rope_rows_of(a);
  const Span sp = VBH_SPAN(parts, static_cast<int64_t>(rows.q + rows.k) * a.dim);
  const int block = static_cast<int>(blockIdx.x);
  const int cut = min(max(a.q().chunks * a.q().walkers - block * kRopeWaves, 0), kRopeWaves);
  for (int d = static_cast<int>(threadIdx.x); d < a.dim; d += kRopeBlock) {
    float q = 0.0f, k = 0.0f;
    for (int v = 0; v < cut * each; ++v) q += sums[v * a.dim + d];
    for (int v = cut * each; v < kRopeWaves * each; ++v) k += sums[v * a.dim + d];
    if (block < rows.q)
      store_any<float, 1, false>(parts + static_cast<int64_t>(block) * a.dim + d, &q, sp);
    if (block >= rows.k_from && block - rows.k_from < rows.k)
      store_any<float, 1, false>(
          parts + static_cast<int64_t>(rows.q + block - rows.k_from) * a.dim + d, &k, sp);
  }
}

// Whether a vector's gradients need sum(dn w u), which has to wait for r, since `dot`,
// sum(dn w x), leaves the range of 32 bits: it is infinite (or not a number), or the vector
// so small that terms of dot may be lost below 2^-149.  Those move mean(dn w u) by less than
// 2^-149 r and du - u mean(dn w u) by that times |u| <= 32: below 2^-24 of a du of 2^-100
// and more while r <= 2^20, where any eps of 2^-40 and more keeps it.
__device__ __forceinline__ bool needs_unit_sum(float dot, float r) {
  return past_range(dot) || r > 0x1p20f;
}

// The wave's share of its tokens, U passes at a time (MORE: more than once); dw: the
// lane's sums.  True if a vector needs_unit_sum: AGAIN goes over the share once more and
// stores such vectors' gradients.  (Apart from the first time, whose registers it leaves
// alone: 16384 tokens of 40 bf16 heads of 128, half pairing, 86.2 us, as without a second
// sum; with it in place 93.)
template <typename T, int V, int U, bool MORE, bool AGAIN, bool ADJ, int WAY, int MEM>
__device__ __forceinline__ bool grad_share(const RopeArgs& a, const RopeSide& side,
                                           const RopeLane& l, int chunk, int first,
                                           float* lds, float (&dw)[V]) {
  const RopeLds parts = rope_lds_of(a, 2 * kGradPasses, kGradPasses);
  float2* table = reinterpret_cast<float2*>(lds);
  float* scratch = lds + parts.table;
  char* rows = reinterpret_cast<char*>(scratch + parts.scratch);
  const Span sx = VBH_SPAN(static_cast<const T*>(side.x), rope_extent(a, side.xs, side.heads));
  const Span sg = VBH_SPAN(static_cast<const T*>(side.g), rope_extent(a, side.gs, side.heads));
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  const int head0 = chunk * (MORE ? side.per_wave : U) * a.tile.per_pass;
  float w[V];
  load_weights<T, V>(a, side, l, w);
  const T* x0 = static_cast<const T*>(side.x);
  const T* g0 = static_cast<const T*>(side.g);
  const int64_t lane_x = (head0 + l.sub) * side.xs[2] + l.at * V;
  const int64_t lane_g = (head0 + l.sub) * side.gs[2] + l.at * V;
  const int64_t x_step = a.tile.per_pass * side.xs[2], g_step = a.tile.per_pass * side.gs[2];
  const int to = (head0 + l.sub) * a.dim + l.at * V, y_step = a.tile.per_pass * a.dim;
  const RopeAngles angles(a);
  bool again = false;

  for (int64_t token = first; token < a.tokens; token += side.walkers) {
    const RopeToken t = rope_token(a, token);
    const double pos = angles.position(a, t);
    const T* from_x = x0 + token_offset(t, side.xs) + lane_x;
    const T* from_g = g0 + token_offset(t, side.gs) + lane_g;
    const RopeOut<T, V, MEM> out(a, side, t.t);
    Turn<V> turn;
    // the share's passes, U at a time
    for (int pass = 0; pass < (MORE ? side.per_wave : U); pass += U) {
      typename Raw<T, V>::type x[U], g[U];
      bool ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // lanes without a vector read their values of the first: no branch keeps the
        // loads apart
        ok[u] = l.live && head0 + (pass + u) * a.tile.per_pass + l.sub < side.heads;
        g[u] = load_any<T, V, MEM != kRopeCached>(
            ok[u] ? from_g + (pass + u) * g_step : g0 + l.at * V, sg);
        x[u] = load_any<T, V, MEM != kRopeCached>(
            ok[u] ? from_x + (pass + u) * x_step : x0 + l.at * V, sx);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // and, with no gradient and r = 0 below, add nothing to the weights' sums
        // (not a number only where the first vector makes them so)
        if (!ok[u]) g[u] = typename Raw<T, V>::type{};
      }
      if (pass == 0) {
        wave_lds_fence();
        angles.make(a, t, pos, table);
        wave_lds_fence();
        make_turn<V, ADJ, WAY>(a, l, table, turn);
      }
      const RopePartners<T, V, U, WAY> partners(a, l, g, rows);
      float dn[U][V], sums[2 * U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float other[V], dot = 0.0f;
        if constexpr (!ADJ) partners.get(g[u], u, other);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float gi = raw_at<T, V>(g[u], i);
          const float gp = ADJ ? raw_at<T, V>(g[u], i ^ 1) : other[i];
          float n = fmaf(gi, turn.c[i], gp * turn.s[i]);
          if (WAY != kRopeWhole && turn.passing[i]) n = gi;
          dn[u][i] = n;
          dot = fmaf(n * w[i], raw_at<T, V>(x[u], i), dot);
        }
        sums[2 * u] = squares<T, V>(x[u]);
        sums[2 * u + 1] = dot;
      }
      vector_sums<2 * U>(a, l, sums, scratch);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float r = ok[u] ? inverse_root(fmaf(sums[2 * u], inv_dim, a.eps)) : 0.0f;
        float mean = sums[2 * u + 1] * r * inv_dim;
        const bool needs = ok[u] && needs_unit_sum(sums[2 * u + 1], r);
        again = again || needs;
        if constexpr (AGAIN) {
          float dot[1] = {0.0f};
#pragma unroll
          for (int i = 0; i < V; ++i)
            dot[0] = fmaf(dn[u][i] * w[i], raw_at<T, V>(x[u], i) * r, dot[0]);
          vector_sums<1>(a, l, dot, scratch);
          mean = dot[0] * inv_dim;
        }
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float unit = raw_at<T, V>(x[u], i) * r;
          if constexpr (!AGAIN) dw[i] = fmaf(dn[u][i], unit, dw[i]);
          // r last: dn r, like dn w x, may leave the range of 32 bits
          o[i] = r * fmaf(dn[u][i], w[i], -unit * mean);
        }
        out.store(to + (pass + u) * y_step, AGAIN ? needs : ok[u], o);
      }
    }
  }
  return again;
}

template <typename T, int V, bool ADJ, int WAY, int MEM>
__global__ __launch_bounds__(kRopeBlock, 4) void qk_norm_rope_grads(const RopeArgs,
                                                                    float* parts) {
  const RopeArgs& a = launch_args();
  extern __shared__ __align__(16) float rope_lds[];
  const int wave = wave_index();
  const RopeWalk walk = rope_walk(a, wave);
  const RopeLane l = rope_lane(a);
  const RopeSide& side = a.side(!walk.is_q);
  float* lds = rope_lds + wave * rope_lds_of(a, 2 * kGradPasses, kGradPasses).all();
  float dw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) dw[i] = 0.0f;
  if (walk.live) {
    bool again;
    if (side.per_wave == 1)
      again = grad_share<T, V, 1, false, false, ADJ, WAY, MEM>(a, side, l, walk.chunk, walk.token,
                                                              lds, dw);
    else if (side.per_wave == kGradPasses)
      again = grad_share<T, V, kGradPasses, false, false, ADJ, WAY, MEM>(a, side, l, walk.chunk,
                                                                        walk.token, lds, dw);
    else
      again = grad_share<T, V, kGradPasses, true, false, ADJ, WAY, MEM>(a, side, l, walk.chunk,
                                                                       walk.token, lds, dw);
    if (__builtin_expect(wave_any(again), 0))
      grad_share<T, V, 1, true, true, ADJ, WAY, MEM>(a, side, l, walk.chunk, walk.token, lds, dw);
  }
  if (parts == nullptr) return;
  __syncthreads();
  if (l.live) {
    float* to = rope_lds + (wave * a.tile.per_pass + l.sub) * a.dim + l.at * V;
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = dw[i];
  }
  __syncthreads();
  write_part(a, rope_lds, a.tile.per_pass, parts);
}

// Pair by pair (rope.h).
template <typename T, int K, bool ADJ>
__global__ __launch_bounds__(kRopeBlock) void qk_norm_rope_value_grads(const RopeArgs a,
                                                                       float* parts) {
  extern __shared__ __align__(16) float rope_lds[];
  const int wave = wave_index();
  float2* table =
      reinterpret_cast<float2*>(rope_lds + wave * rope_lds_of(a, 0, 0).table);
  const RopeLane l = rope_lane(a);
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  float dw[2 * K];
#pragma unroll
  for (int k = 0; k < 2 * K; ++k) dw[k] = 0.0f;
  const RopeWalk walk = rope_walk(a, wave);
  const RopeSide& side = a.side(!walk.is_q);
  const int head = walk.chunk * a.tile.per_pass + l.sub;

  const RopeAngles angles(a);
  for (int64_t token = walk.live ? walk.token : a.tokens; token < a.tokens;
       token += side.walkers) {
    const RopeToken t = rope_token(a, token);
    const bool ok = l.live && head < side.heads;
    const Span sx = VBH_SPAN(static_cast<const T*>(side.x), rope_extent(a, side.xs, side.heads));
    const Span sg = VBH_SPAN(static_cast<const T*>(side.g), rope_extent(a, side.gs, side.heads));
    const Span sy = VBH_SPAN(static_cast<T*>(side.y), a.tokens * side.heads * a.dim);
    const T* x = static_cast<const T*>(side.x) + token_offset(t, side.xs) + head * side.xs[2];
    const T* g = static_cast<const T*>(side.g) + token_offset(t, side.gs) + head * side.gs[2];
    T* y = static_cast<T*>(side.y) + (t.t * side.heads + head) * a.dim;
    wave_lds_fence();
    angles.make(a, t, angles.position(a, t), table);
    wave_lds_fence();
    float xa[K], xb[K], na[K], nb[K], sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const RopePair r = rope_pair<ADJ>(a, l, k);
      const bool has_a = ok && r.has_a, has_b = ok && r.has_b;
      xa[k] = load_value<T>(x + r.a, has_a, sx);
      xb[k] = load_value<T>(x + r.b, has_b, sx);
      na[k] = load_value<T>(g + r.a, has_a, sg);
      nb[k] = load_value<T>(g + r.b, has_b, sg);
      if (has_a && r.p >= 0) {
        const float2 cs = table[table_place(r.p)];
        const float ga = na[k], gb = nb[k];
        na[k] = fmaf(ga, cs.x, -gb * cs.y);
        nb[k] = fmaf(gb, cs.x, ga * cs.y);
      }
      sums[0] = fmaf(xa[k], xa[k], fmaf(xb[k], xb[k], sums[0]));
      if (has_a) sums[1] = fmaf(na[k] * load_weight<T>(a, side, r.a), xa[k], sums[1]);
      if (has_b) sums[1] = fmaf(nb[k] * load_weight<T>(a, side, r.b), xb[k], sums[1]);
    }
    vector_sums<2>(a, l, sums, nullptr);
    const float size = inverse_root(fmaf(sums[0], inv_dim, a.eps));
    float mean = sums[1] * size * inv_dim;
    const bool needs = ok && needs_unit_sum(sums[1], size);
    if (__builtin_expect(wave_any(needs), 0)) {
      float dot[1] = {0.0f};
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const RopePair r = rope_pair<ADJ>(a, l, k);
        if (ok && r.has_a)
          dot[0] = fmaf(na[k] * load_weight<T>(a, side, r.a), xa[k] * size, dot[0]);
        if (ok && r.has_b)
          dot[0] = fmaf(nb[k] * load_weight<T>(a, side, r.b), xb[k] * size, dot[0]);
      }
      vector_sums<1>(a, l, dot, nullptr);
      if (needs) mean = dot[0] * inv_dim;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const RopePair r = rope_pair<ADJ>(a, l, k);
      const float ua = xa[k] * size, ub = xb[k] * size;
      if (ok && r.has_a) {
        const float o = size * fmaf(na[k], load_weight<T>(a, side, r.a), -ua * mean);
        store_any<T, 1>(y + r.a, &o, sy);
        dw[2 * k] = fmaf(na[k], ua, dw[2 * k]);
      }
      if (ok && r.has_b) {
        const float o = size * fmaf(nb[k], load_weight<T>(a, side, r.b), -ub * mean);
        store_any<T, 1>(y + r.b, &o, sy);
        dw[2 * k + 1] = fmaf(nb[k], ub, dw[2 * k + 1]);
      }
    }
  }
  if (parts == nullptr) return;
  __syncthreads();
  float* to = rope_lds + (wave * a.tile.per_pass + l.sub) * a.dim;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const RopePair r = rope_pair<ADJ>(a, l, k);
    if (r.has_a) to[r.a] = dw[2 * k];
    if (r.has_b) to[r.b] = dw[2 * k + 1];
  }
  __syncthreads();
  write_part(a, rope_lds, a.tile.per_pass, parts);
}

// Sums over the rows of parts: a workgroup for 16 values of a side, four to a lane
// and 16 lines of lanes to a wave, so that a thousand rows take one round of loads.
// Lines are added up through the wave, then waves through the LDS, in order.
constexpr int kSumCols = 16;
constexpr int kSumWaves = 16;
constexpr int kSumLines = 16 * kSumWaves;

template <typename W>
__global__ __launch_bounds__(kSumWaves* kWave) void qk_weight_grads(const float* parts, int q_rows,
                                                                    int k_rows, int dim, W* dq,
                                                                    W* dk) {
  __shared__ float sums[kSumWaves][kSumCols];
  const bool is_q = blockIdx.y == 0;
  W* out = is_q ? dq : dk;
  if (out == nullptr) return;
  const Span sp = VBH_SPAN(parts, static_cast<int64_t>(q_rows + k_rows) * dim);
  const Span so = VBH_SPAN(out, dim);
  const int wave = wave_index(), lane = wave_lane();
  const int d = static_cast<int>(blockIdx.x) * kSumCols + (lane / 16) * 4;
  const int rows = is_q ? q_rows : k_rows;
  const float* from = parts + static_cast<int64_t>(is_q ? 0 : q_rows) * dim;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int r = wave * 16 + lane % 16; r < rows; r += 4 * kSumLines) {
    // four rows' loads in flight; rows behind the last are the first of them again
    const float* row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int rr = r + j * kSumLines;
      row[j] = from + static_cast<int64_t>(rr < rows ? rr : r) * dim + d;
    }
    float x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = 0.0f;
      if (dim % 4 == 0 && d < dim) {
        const typename Raw<float, 4>::type y = load_any<float, 4, false>(row[j], sp);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j][i] = y[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < dim) x[j][i] = load_any<float, 1, false>(row[j] + i, sp);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += r + j * kSumLines < rows ? x[j][i] : 0.0f;
    }
  }
  wave_sums<4>(v, 4);
  if (lane % 16 == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][lane / 4 + i] = v[i];
  }
  __syncthreads();
  const int c = static_cast<int>(threadIdx.x), to = static_cast<int>(blockIdx.x) * kSumCols + c;
  if (c >= kSumCols || to >= dim) return;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kSumWaves; ++i) sum += sums[i][c];
  store_any<W, 1, false>(out + to, &sum, so);
}

// Waves of a launch, whatever the kernel: as many as the card holds at once of the 16-bit
// ones with 16-byte accesses, 4 to a SIMD (with single passes only, 6 or 8 fit, and 8192
// tokens of 40 bf16 heads of 128 take 57.6 and 87.9 us against 48.3).  5 to 8 would fit of
// those that hold 59 to 92 registers (accesses of 2 values, one pair to a lane, fp32 with
// adjacent pairs); of that of eight pairs to a lane 2 or 3 do (136 to 168 registers in
// fp32, 184 to 200 in 16 bits), and the others wait for a second round.  No counts of
// their own were tried.  kGradMany: passes beyond which a wave takes more than one of a
// token's, whose angles it then makes once.  Up to 4 of them where a token's angles take one
// round of the lanes and vectors lie over a power of two of them without a gap, 8 otherwise.
// MI355X, 16384 tokens of 40 bf16 heads, us at 2 / 4 / 8: of 128 87.4 / 87.1 / 87.6 (65536
// tokens 371 / 367 / 378), 192 94 / 85 / 79, 256 104 / 92 / 91 (both 8192 tokens),
// 100 113 / 109 / 99, 50 97 / 97 / 85, 96 75.6 / 73.9 / 71.8.
constexpr int64_t kGradWaves = 4096;
constexpr int64_t kGradMany = 4 * kGradWaves;
constexpr int kGradShare = 8;

// rope_shape, and the walkers of each side: waves in proportion to its work, no more
// than it has tokens, and none that would only share the last turn of the others.
void grad_shape(RopeArgs& a, int dt, bool adjacent) {
  rope_shape(a, dt, adjacent, true, kGradMany, kGradPasses, kGradShare, true);
  auto work = [&](const RopeSide& s) { return int64_t(s.chunks) * (s.per_wave + 2); };
  const int64_t all = work(a.q()) + work(a.k());
  for (RopeSide* s : {&a.q(), &a.k()}) {
    s->walkers = 0;
    if (s->chunks == 0 || a.tokens == 0) continue;
    const int64_t most =
        std::min(a.tokens, std::max<int64_t>(kGradWaves * (s->per_wave + 2) / all, 1));
    const int64_t turns = (a.tokens + most - 1) / most;
    s->walkers = static_cast<int>((a.tokens + turns - 1) / turns);
  }
}

}  // namespace

int64_t rope_bwd_part_floats(const RopeArgs& args, int dt, bool adjacent) {
  RopeArgs a = args;
  grad_shape(a, dt, adjacent);
  const RopeRows rows = rope_rows_of(a);
  return int64_t(rows.q + rows.k) * a.dim;
}

hipError_t launch_qk_norm_rope_bwd(const RopeArgs& args, int dt, bool adjacent, void* dq_weight,
                                   void* dk_weight, float* parts, hipStream_t s) {
  RopeArgs a = args;
  grad_shape(a, dt, adjacent);
  const RopeTile& t = a.tile;
  const RopeRows rows = rope_rows_of(a);
  const bool whole = 2 * a.n_freq == a.dim && (adjacent || a.n_freq % t.v == 0);
  const bool sums = dq_weight != nullptr || dk_weight != nullptr;
  const int64_t bytes =
      a.tokens * (a.q().heads + a.k().heads) * a.dim * (dt == kF32 ? 4 : 2);
  const int waves = a.q().chunks * a.q().walkers + a.k().chunks * a.k().walkers;
  hipError_t err = hipSuccess;
  if (waves > 0) {
    const size_t row_sums = sums ? size_t(kRopeWaves) * t.per_pass * a.dim : 0;
    auto go = [&](auto kernel, size_t floats) {
      launch_kernel(kernel, dim3((waves + kRopeWaves - 1) / kRopeWaves), dim3(kRopeBlock),
                    static_cast<unsigned>(std::max(floats, row_sums) * sizeof(float)), s, a,
                    sums ? parts : nullptr);
      err = hipGetLastError();
    };
    dispatch_float_type(dt, [&](auto tt) {
      using T = typename decltype(tt)::type;
      constexpr int VN = Vec<T>::n;
      dispatch_bool(adjacent, [&](auto ac) {
        constexpr bool A = decltype(ac)::value;
        if (t.v == 1) {
          const size_t floats = size_t(kRopeWaves) * rope_lds_of(a, 0, 0).table;
          if ((a.dim + 1) / 2 <= kWave) go(qk_norm_rope_value_grads<T, 1, A>, floats);
          else go(qk_norm_rope_value_grads<T, kRopePairs, A>, floats);
          return;
        }
        const size_t floats =
            size_t(kRopeWaves) * rope_lds_of(a, 2 * kGradPasses, kGradPasses).all();
        auto grads = [&](auto mc) {
          constexpr int M = decltype(mc)::value;
          if (t.v == VN && whole) return go(qk_norm_rope_grads<T, VN, A, kRopeWhole, M>, floats);
          dispatch_bool(a.gather != 0, [&](auto gc) {
            constexpr int W = decltype(gc)::value && !A ? kRopeGather : kRopeHalves;
            if (t.v == VN) go(qk_norm_rope_grads<T, VN, A, W, M>, floats);
            else if (VN == 8 && t.v == 4) go(qk_norm_rope_grads<T, 4, A, W, M>, floats);
            else go(qk_norm_rope_grads<T, 2, A, W, M>, floats);
          });
        };
        dispatch_rope_mem(rope_mem(2 * bytes, bytes), grads);
      });
    });
  }
  if (err != hipSuccess || !sums) return err;
  auto sum = [&](auto tag) {
    using W = typename decltype(tag)::type;
    launch_kernel(qk_weight_grads<W>, dim3((a.dim + kSumCols - 1) / kSumCols, 2),
                  dim3(kSumWaves * kWave), 0, s, parts, rows.q, rows.k, a.dim,
                  static_cast<W*>(dq_weight), static_cast<W*>(dk_weight));
    err = hipGetLastError();
  };
  if (a.w_f32) sum(TypeTag<float>{});
  else dispatch_float_type(dt, sum);
  return err;
}

}  // namespace vbh
