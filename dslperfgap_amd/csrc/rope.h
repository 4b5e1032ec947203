// What the rotation kernels (rope.hip, rope_bwd.hip) share: their arguments, a
// lane's place among a token's heads, and the angles.
//
// A token has H = q_heads + k_heads vectors of D values.  A vector belongs to a
// group of lanes (a power of two up to 64); a lane holds two pieces of it, A and
// B, of V values each, chosen so that both members of every pair are its own:
//   half pairing:      A[i] turns with B[i] (B lies n_freq values behind A)
//   adjacent pairing:  A[2i] with A[2i+1], B[2i] with B[2i+1] (B lies D / 2 behind
//                      A, so that the loads run over the vector as in the other)
// and nothing crosses lanes but the norm's sums.  The values that do not turn are
// paired the same way among themselves.  A wave holds 64 / G vectors of one
// token at a time, heads [chunk * 64 / G, ...) for its whole life.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vbh_device.h"
#include "vbh_launch.h"

namespace vbh {

constexpr int kRopeWaves = 4;  // waves per workgroup
constexpr int kRopeBlock = kRopeWaves * kWave;

// A lane's vector: head `head` of the token's q_heads + k_heads, place `at` in the
// group.
struct RopeLane {
  int head, at;
  bool live, is_q;
};

__device__ __forceinline__ RopeLane rope_lane(const RopeArgs& a, int chunk) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  RopeLane l;
  l.head = chunk * (kWave >> a.group_log2) + (lane >> a.group_log2);
  l.at = lane & ((1 << a.group_log2) - 1);
  l.live = l.head < a.q.heads + a.k.heads;
  l.is_q = l.head < a.q.heads;
  return l;
}

// The lane's k-th pieces: places of A and B in the vector, its first pair slot,
// and which of them there are.
struct RopePiece {
  int a, b, slot;
  bool has_a, has_b;
};

template <int V, bool ADJ>
__device__ __forceinline__ RopePiece rope_piece(const RopeArgs& a, const RopeLane& l, int k) {
  RopePiece p;
  p.slot = (l.at + k * kWave) * V;
  if constexpr (ADJ && V == 1) {
    p.a = 2 * p.slot;
    p.b = p.a + 1;
  } else if constexpr (ADJ) {
    p.a = p.slot;
    p.b = a.slots + p.slot;
  } else {
    const bool turns = p.slot < a.n_freq;
    p.a = turns ? p.slot : a.n_freq + p.slot;
    p.b = p.a + (turns ? a.n_freq : a.slots - a.n_freq);
  }
  p.has_a = l.live && p.slot < a.slots;
  p.has_b = p.has_a && (V > 1 || p.b < a.dim);
  return p;
}

// Pair of the i-th (A, B) values of a piece (half pairing) or of the i-th pair of
// its 2 V values (adjacent pairing: V / 2 pairs in A, then V / 2 in B).
template <int V, bool ADJ>
__device__ __forceinline__ int rope_pair(const RopeArgs& a, const RopePiece& p, int i) {
  if constexpr (ADJ && V > 1)
    return (p.slot >> 1) + (i < V / 2 ? i : (a.slots >> 1) + i - V / 2);
  else
    return p.slot + i;
}

__device__ __forceinline__ Span pick_span(bool first, const Span& a, const Span& b) {
  return first ? a : b;
}

// n consecutive (cos, sin) of the table (16-byte aligned where n is even)
template <int N>
__device__ __forceinline__ void read_angles(const float2* table, float* c, float* s) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float4 v = *reinterpret_cast<const float4*>(table + i);
      c[i] = v.x;
      s[i] = v.y;
      c[i + 1] = v.z;
      s[i + 1] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = table[i].x;
      s[i] = table[i].y;
    }
  }
}

// The V pairs' (cos, sin) of a piece, in rope_pair's order.
template <int V, bool ADJ>
__device__ __forceinline__ void piece_angles(const RopeArgs& a, const RopePiece& p,
                                             const float2* table, float (&c)[V], float (&s)[V]) {
  if constexpr (ADJ && V > 1) {
    read_angles<V / 2>(table + (p.slot >> 1), c, s);
    read_angles<V / 2>(table + (a.slots >> 1) + (p.slot >> 1), c + V / 2, s + V / 2);
  } else {
    read_angles<V>(table + p.slot, c, s);
  }
}

// The two values of pair i among a piece's 2 V values (A first).
template <int V, bool ADJ>
__device__ __forceinline__ void pair_at(int i, int& first, int& second) {
  first = ADJ && V > 1 ? 2 * i : i;
  second = ADJ && V > 1 ? 2 * i + 1 : V + i;
}

template <typename T, int V>
__device__ __forceinline__ void load_piece(const T* x, const RopePiece& p,
                                           typename Raw<T, V>::type& ra,
                                           typename Raw<T, V>::type& rb, const Span& s) {
  ra = p.has_a ? load_any<T, V>(x + p.a, s) : typename Raw<T, V>::type{};
  rb = p.has_b ? load_any<T, V>(x + p.b, s) : typename Raw<T, V>::type{};
}

// A piece's 2 V weights (ones without a weight), widened.
template <typename T, int V>
__device__ __forceinline__ void load_weights(const RopeArgs& a, const RopeLane& l,
                                             const RopePiece& p, float (&w)[2 * V]) {
  const void* from = l.is_q ? a.q.w : a.k.w;
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) w[i] = 1.0f;
  if (from == nullptr || !p.has_a) return;
  auto widen = [&](auto tag) {
    using W = typename decltype(tag)::type;
    const W* wp = static_cast<const W*>(from);
    const Span s = VBH_SPAN(wp, a.dim);
    const typename Raw<W, V>::type wa = load_any<W, V, false>(wp + p.a, s);
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = raw_at<W, V>(wa, i);
    if (!p.has_b) return;
    const typename Raw<W, V>::type wb = load_any<W, V, false>(wp + p.b, s);
#pragma unroll
    for (int i = 0; i < V; ++i) w[V + i] = raw_at<W, V>(wb, i);
  };
  if (a.w_f32) widen(TypeTag<float>{});
  else widen(TypeTag<T>{});
}

// Values of an operand with strides `st` (for Spans).
__device__ __forceinline__ int64_t rope_extent(const RopeArgs& a, const int64_t (&st)[3],
                                               int heads) {
  return heads > 0 ? (a.batch - 1) * st[0] + (a.seq - 1) * st[1] + (heads - 1) * st[2] + a.dim : 0;
}

// Sums of N values over each group of 2^group_log2 lanes, in every lane of it.
template <int N>
__device__ __forceinline__ void group_sums(float (&v)[N], int group_log2) {
  const int width = 1 << group_log2;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_allreduce<Sum>(v[i], width);
}

// 1 / sqrt(m) for m >= 0; v_rsq_f32 takes no subnormal operand.
__device__ __forceinline__ float inverse_root(float m) {
  const bool tiny = m < 0x1p-96f;
  return __builtin_amdgcn_rsqf(tiny ? m * 0x1p96f : m) * (tiny ? 0x1p48f : 1.0f);
}

// What one wave wrote to its part of the LDS is there for all of its lanes (the
// wave's LDS accesses stay in order; this keeps the compiler to it).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------------------
// angles
// ---------------------------------------------------------------------------

// sin and cos of 2 pi f, |f| <= 1/2 turn: f is reduced to r, at most an eighth of
// a turn, in 64 bits, and the Taylor series around 0 are summed in 32: the first
// terms left out, x^11 / 11! and x^12 / 12! at x = pi / 4, are 1.8e-9 and 1.2e-10.
__device__ __forceinline__ float2 cos_sin_turns(double f) {
  const double k = __builtin_rint(f * 4.0);
  const float x = static_cast<float>((f - 0.25 * k) * 6.283185307179586);
  const int quarter = static_cast<int>(k);
  const float x2 = x * x;
  float s = fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(x2, s, 8.3333333e-3f);
  s = fmaf(x2, s, -0.16666667f);
  s = fmaf(x2 * x, s, x);
  float c = fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(x2, c, -1.3888889e-3f);
  c = fmaf(x2, c, 4.1666667e-2f);
  c = fmaf(x2, c, -0.5f);
  c = fmaf(x2, c, 1.0f);
  const bool swap = (quarter & 1) != 0;
  const float co = swap ? s : c, si = swap ? c : s;
  // quarter 1: (cos, sin) = (-s, c); 2: (-c, -s); 3: (s, -c)
  return make_float2((quarter + 1) & 2 ? -co : co, quarter & 2 ? -si : si);
}

__device__ __forceinline__ double load_position(const RopeArgs& a, int64_t at, const Span& s) {
  if (a.pos_dt == kI64) {
    const int64_t* p = static_cast<const int64_t*>(a.pos) + at;
    return VBH_IN_SPAN(s, p, 8) ? static_cast<double>(*p) : 0.0;
  }
  if (a.pos_dt == kI32) {
    const int32_t* p = static_cast<const int32_t*>(a.pos) + at;
    return VBH_IN_SPAN(s, p, 4) ? static_cast<double>(*p) : 0.0;
  }
  const float* p = static_cast<const float*>(a.pos) + at;
  return VBH_IN_SPAN(s, p, 4) ? static_cast<double>(*p) : 0.0;
}

// Turns per unit of position of pair p (0 where the pair passes).
__device__ __forceinline__ double load_turns(const RopeArgs& a, int p, const Span& s) {
  constexpr double kInvTwoPi = 0.15915494309189535;
  if (p >= a.n_freq) return 0.0;
  if (a.f64_freq) {
    const double* f = static_cast<const double*>(a.freq) + p;
    return VBH_IN_SPAN(s, f, 8) ? *f * kInvTwoPi : 0.0;
  }
  const float* f = static_cast<const float*>(a.freq) + p;
  return VBH_IN_SPAN(s, f, 4) ? static_cast<double>(*f) * kInvTwoPi : 0.0;
}

// Position axis of pair p.
__device__ __forceinline__ int axis_of(const RopeArgs& a, int p) {
  if (a.axes == 1) return 0;
  if (a.section_order == 0) {  // ends[i]: first pair behind axis i's block
    int ax = 0;
#pragma unroll
    for (int i = 0; i < kRopeMaxAxes - 1; ++i) ax += i + 1 < a.axes && p >= a.ends[i] ? 1 : 0;
    return ax;
  }
  const int ax = p % a.axes;
  int end = a.ends[0];  // ends[i]: axes * sections[i]
#pragma unroll
  for (int i = 1; i < kRopeMaxAxes; ++i) end = ax == i ? a.ends[i] : end;
  return p < end ? ax : 0;
}

// The wave's table of (cos, sin) * scale of `slots` pairs for each of U tokens, in
// its own part of the LDS: every lane makes one pair's at a time, however many
// heads then read it.  Pairs that pass are (1, 0).
template <int U>
__device__ __forceinline__ void make_angles(const RopeArgs& a, int64_t t0, int b0, int s0,
                                            float2* table) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const Span sf = VBH_SPAN(static_cast<const char*>(a.freq),
                           static_cast<int64_t>(a.n_freq) * (a.f64_freq ? 8 : 4));
  const Span sp = VBH_SPAN(static_cast<const char*>(a.pos),
                           a.pos_elems * (a.pos_dt == kI64 ? 8 : 4));
  // slot_log2: slots rounded up to a power of two, at most the wave
  const int per = kWave >> a.slot_log2;  // tokens at a time
  const int du = lane >> a.slot_log2;
  for (int p = lane & ((1 << a.slot_log2) - 1); p < a.slots; p += kWave) {
    const double turns = load_turns(a, p, sf);
    const int64_t from = axis_of(a, p) * a.pos_stride[0];
    for (int u = du; u < U; u += per) {
      int b = b0, s = s0 + u;
      while (s >= a.seq) {
        s -= a.seq;
        ++b;
      }
      if (t0 + u >= a.tokens) break;
      float2 cs = make_float2(1.0f, 0.0f);
      if (p < a.n_freq) {
        const double pos =
            load_position(a, from + b * a.pos_stride[1] + s * a.pos_stride[2], sp);
        const double f = pos * turns;
        cs = cos_sin_turns(f - __builtin_rint(f));
        cs.x *= a.scale;
        cs.y *= a.sin_scale;
      }
      table[u * a.slots + p] = cs;
    }
  }
}

}  // namespace vbh
