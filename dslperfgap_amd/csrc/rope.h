// What the rotation kernels (rope.hip, rope_bwd.hip) share.
//
// A token has q_heads + k_heads vectors of D values.  A wave takes a share of one
// token's queries or of its keys, so that the angles are made once (one sincos per
// lane for 64 pairs, through the LDS) for up to kRopePasses passes over vectors (the norm's
// backward: up to kGradShare, kGradPasses of them at a time).  In a pass
// the wave holds `per_pass` vectors side by side, each lane V consecutive values:
// the accesses of a pass run over memory without gaps wherever the heads do.  (Both
// members of every pair in one lane, as two pieces of half the vector each, costs no
// exchange, but pieces of less than a 128-byte line cost more: on MI355X 38 us against
// 27 for 16384 tokens of 40 bf16 heads of 64.)
//   adjacent pairing: a lane's values pair among themselves
//   half pairing:     the partners lie in other lanes of the vector's, n_freq / V
//                     away, whose 16 bytes come over the LDS crossbar as they are
//                     stored; both lanes then widen both vectors (RopePartner)
// Per value y_i = (x_i r) C_i + (x_partner r) S_i: the cosines and sines, their signs,
// the scale and the weights meet in C and S once per wave, so that the norm adds
// its sum of squares and one product per value, two in half pairing.  (One product
// with r at the end would do, but x_i C_i may pass the range of 32 bits where y_i
// does not.)
//
// Vectors that no lane access of 2 values or more fits (odd sizes, more than 64
// lanes) go pair by pair: a lane holds both members of a pair (rope_values,
// qk_norm_rope_value_grads).
#pragma once

#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "vbh_device.h"
#include "vbh_launch.h"

namespace vbh {

constexpr int kCacheSc1 = 1 << 4;  // cache-policy operand: device scope
constexpr int kRopeWaves = 4;  // waves per workgroup
constexpr int kRopeBlock = kRopeWaves * kWave;
constexpr int kRopePairs = 8;  // pairs of a lane that goes pair by pair
constexpr int kRopePasses = 4; // passes of a wave's share in rope_rows, at most

// How a launch treats memory (rope_mem): kRopeCached, kRopeOnce: nontemporal loads,
// kRopeStream: nontemporal loads and stores.  All write through the L2 at device scope,
// so that nothing is left to write back when the kernel ends: MI355X, us without / with:
// 16384 tokens of 40 bf16 heads of 128, rotation 52.1 / 50.5, backward 91.3 / 86.5;
// 8192 tokens, norm and rotation 29.5 / 28.9; 32768, rotation (kRopeStream) 107.9 / 105.3.
enum RopeMem : int { kRopeCached = 0, kRopeOnce = 1, kRopeStream = 2 };

// What a launch reads and writes, against the 256 MiB cache in front of the memory.
// MI355X, tokens of 40 bf16 heads of 128, half pairing, three sets of inputs in turn, us as
// kRopeCached / kRopeOnce / kRopeStream (backward: twice as much read as written):
//   tokens, MB written    rotation              norm and rotation     backward
//   2048, 21               9.2 /  9.2 /  9.5     9.8 / 10.2 / 10.3    20.7 / 22.0 / 22.2
//   4096, 42              14.8 / 16.1 / 17.2    15.8 / 17.7 / 18.6    31.7 / 31.9 / 33.0
//   8192, 84              28.1 / 28.0 / 30.1    30.6 / 30.2 / 31.8    50.7 / 49.1 / 52.4
//   16384, 168            59.9 / 50.4 / 54.8    60.8 / 54.3 / 57.5   102.5 / 85.9 / 93.6
//   32768, 336           117.4 /106.6 /104.8   114.0 /110.6 /109.4   197.1 /188.4 /180.3
constexpr int64_t kRopeCachedBytes = int64_t(128) << 20;  // read and written
constexpr int64_t kRopeOnceBytes = int64_t(224) << 20;    // written
inline RopeMem rope_mem(int64_t read, int64_t written) {
  if (written > kRopeOnceBytes) return kRopeStream;
  return read + written > kRopeCachedBytes ? kRopeOnce : kRopeCached;
}
template <typename Fn>
void dispatch_rope_mem(RopeMem m, Fn&& fn) {
  if (m == kRopeCached) fn(std::integral_constant<int, kRopeCached>{});
  else if (m == kRopeOnce) fn(std::integral_constant<int, kRopeOnce>{});
  else fn(std::integral_constant<int, kRopeStream>{});
}

constexpr int kRopeScratch = 128;  // floats per sum: 64 lanes, lines of 4

// A wave's part of the LDS, in floats (whole 16-byte vectors): its table of angles, the
// scratch of `sums` sums where vectors are no power of two of lanes, and where a.gather
// the vectors of `passes` passes.
struct RopeLds {
  int table, scratch, rows;
  __host__ __device__ int all() const { return table + scratch + rows; }
};
__host__ __device__ inline RopeLds rope_lds_of(const RopeArgs& a, int sums, int passes) {
  RopeLds r;
  r.table = (2 * a.n_freq + 15) & ~15;  // table_place stays in runs of 8 pairs
  r.scratch = a.tile.lanes_log2 < 0 ? sums * kRopeScratch : 0;
  r.rows = a.gather ? passes * (kWave * 16 / 4) : 0;
  return r;
}

// Values of an operand with strides `st` (for Spans).
__device__ __forceinline__ int64_t rope_extent(const RopeArgs& a, const int64_t (&st)[3],
                                               int heads) {
  return heads > 0 ? (a.batch - 1) * st[0] + (a.seq - 1) * st[1] + (heads - 1) * st[2] + a.dim : 0;
}

// 1 / sqrt(m) for m >= 0; v_rsq_f32 takes no subnormal operand.
__device__ __forceinline__ float inverse_root(float m) {
  const bool tiny = m < 0x1p-96f;
  return __builtin_amdgcn_rsqf(tiny ? m * 0x1p96f : m) * (tiny ? 0x1p48f : 1.0f);
}

// Infinite or not a number.
__device__ __forceinline__ bool past_range(float x) { return !(fabsf(x) <= 0x1.fffffep127f); }

// True in every lane where it is in one of the wave's.
__device__ __forceinline__ bool wave_any(bool b) { return __ballot(b) != 0; }

// What one wave wrote to its part of the LDS is there for all of its lanes (the
// wave's LDS accesses stay in order; this keeps the compiler to it).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int wave_lane() {
  return static_cast<int>(threadIdx.x) & (kWave - 1);
}
__device__ __forceinline__ int wave_index() {
  return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
}

// The kernel's RopeArgs (its first parameter) where the launch left them: scalar
// loads from there, a side's by its number.  Read through the parameter itself, both
// sides' fields are loaded ahead of every choice between them, and over a hundred of
// the backward's scalars spill.
__device__ __forceinline__ const RopeArgs& launch_args() {
  return *reinterpret_cast<const RopeArgs*>(
      (const void*)__builtin_amdgcn_kernarg_segment_ptr());
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

// Turns per unit of position of pair p.
__device__ __forceinline__ double load_turns(const RopeArgs& a, int p, const Span& s) {
  constexpr double kInvTwoPi = 0.15915494309189535;
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

// Where token t lies: element offsets from its batch and place in it.
struct RopeToken {
  int64_t t;
  int b, s;
};
__device__ __forceinline__ RopeToken rope_token(const RopeArgs& a, int64_t t) {
  RopeToken r{t, 0, static_cast<int>(t)};
  if (a.batch > 1) {
    r.b = static_cast<int>(static_cast<uint32_t>(t) / static_cast<uint32_t>(a.seq));
    r.s = static_cast<int>(t) - r.b * a.seq;
  }
  return r;
}
__device__ __forceinline__ int64_t token_offset(const RopeToken& t, const int64_t (&st)[3]) {
  return t.b * st[0] + t.s * st[1];
}

// Place of pair p in a wave's table of float2, p and p + 1 side by side for even p.
// Lanes read whole runs of pairs, 64 bytes apart at 8 each; the exchange of 16-byte
// words within 64 bytes, another in each 256, lets 16 of them read at once without
// bank conflicts.
__device__ __forceinline__ int table_place(int p) {
  const int word = p >> 1;
  return ((word ^ ((word >> 4) & 3)) << 1) | (p & 1);
}
// N pairs from p on (even where N is).
template <int N>
__device__ __forceinline__ void read_turns(const float2* table, int p, float (&c)[N],
                                           float (&s)[N]) {
  if constexpr (N == 1) {
    const float2 v = table[table_place(p)];
    c[0] = v.x;
    s[0] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float4 v = *reinterpret_cast<const float4*>(table + table_place(p + i));
      c[i] = v.x;
      s[i] = v.y;
      c[i + 1] = v.z;
      s[i + 1] = v.w;
    }
  }
}

// (cos, sin) * scale of pairs lane, lane + 64, ... of a token, one lane each, into
// the wave's table.  What the first of them needs of memory is loaded by itself, so
// that a wave that walks over tokens may ask for it ahead of its other loads, which
// return in order.
struct RopeAngles {
  double turns;    // per unit of position, of pair `lane`
  int64_t axis_at; // its axis's offset among the positions
  Span sf, sp;
  __device__ __forceinline__ explicit RopeAngles(const RopeArgs& a) {
    sf = VBH_SPAN(static_cast<const char*>(a.freq),
                  static_cast<int64_t>(a.n_freq) * (a.f64_freq ? 8 : 4));
    sp = VBH_SPAN(static_cast<const char*>(a.pos), a.pos_elems * (a.pos_dt == kI64 ? 8 : 4));
    const int p = min(wave_lane(), a.n_freq - 1);
    turns = load_turns(a, p, sf);
    axis_at = axis_of(a, p) * a.pos_stride[0];
  }
  __device__ __forceinline__ double position(const RopeArgs& a, const RopeToken& t) const {
    return load_position(a, axis_at + t.b * a.pos_stride[1] + t.s * a.pos_stride[2], sp);
  }
  __device__ __forceinline__ void put(const RopeArgs& a, float2* table, int p, double f) const {
    float2 cs = cos_sin_turns(f - __builtin_rint(f));
    cs.x *= a.scale;
    cs.y *= a.sin_scale;
    table[table_place(p)] = cs;
  }
  __device__ __forceinline__ void make(const RopeArgs& a, const RopeToken& t, double pos,
                                       float2* table) const {
    if (wave_lane() < a.n_freq) put(a, table, wave_lane(), pos * turns);
    const int64_t at = t.b * a.pos_stride[1] + t.s * a.pos_stride[2];
    for (int p = wave_lane() + kWave; p < a.n_freq; p += kWave)
      put(a, table, p, load_position(a, axis_of(a, p) * a.pos_stride[0] + at, sp) *
                           load_turns(a, p, sf));
  }
};

// ---------------------------------------------------------------------------
// passes
// ---------------------------------------------------------------------------

// A lane's place: vector `sub` of the pass, access `at` of it (the last one's for
// lanes behind it, which are not live).
struct RopeLane {
  int sub, at;
  bool live;
};
__device__ __forceinline__ RopeLane rope_lane(const RopeArgs& a) {
  const int lane = wave_lane();
  RopeLane l;
  l.sub = a.tile.lanes_log2 >= 0 ? lane >> a.tile.lanes_log2 : small_quotient(lane, a.tile.lanes);
  const int at = lane - l.sub * a.tile.lanes;
  l.live = l.sub < a.tile.per_pass && at < a.tile.accesses;
  l.at = min(at, a.tile.accesses - 1);
  return l;
}

// Where the partners of a lane's values are (half pairing), by launch.
//   kRopeWhole: all values turn and n_freq is a multiple of V: the whole access has its
//   partners in one lane.
//   kRopeHalves: some values pass (their own partners), or n_freq is a multiple of V / 2
//   only: each half of the access has its partners in one lane, in its own half or,
//   where n_freq is an odd number of halves, in the other (crossed).
//   kRopeGather: any n_freq; the vectors go through the LDS and every value is read by
//   itself.
// Adjacent pairing: kRopeWhole, or kRopeHalves where some values pass.
enum RopeWay : int { kRopeWhole = 0, kRopeHalves = 1, kRopeGather = 2 };
template <int V>
struct RopePartner {
  int lane[2];
  bool crossed;  // of the launch
};
template <int V, int WAY>
__device__ __forceinline__ RopePartner<V> rope_partner(const RopeArgs& a, const RopeLane& l) {
  RopePartner<V> p;
  const int first_lane = l.sub * a.tile.lanes;
  if constexpr (WAY == kRopeWhole) {
    const int away = a.n_freq / V;
    p.lane[0] = p.lane[1] = first_lane + (l.at < away ? l.at + away : l.at - away);
    p.crossed = false;
  } else {
    const int away = a.n_freq / (V / 2);  // halves
    p.crossed = (away & 1) != 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mine = 2 * l.at + h;
      const int theirs = mine < away ? mine + away : mine < 2 * away ? mine - away : mine;
      p.lane[h] = first_lane + (theirs >> 1);
    }
  }
  return p;
}

// The place of value e's partner in its vector (its own where it passes).
__device__ __forceinline__ int partner_of(const RopeArgs& a, int e) {
  return e < a.n_freq ? e + a.n_freq : e < 2 * a.n_freq ? e - a.n_freq : e;
}

// The partners of U passes' accesses, widened one pass at a time.  `rows`: where
// a.gather, kRopeRow * U bytes of the wave's own.
constexpr int kRopeRow = kWave * 16;  // rope_lds_of
template <typename T, int V, int U, int WAY>
struct RopePartners {
  RopePartner<V> p;
  const T* rows;
  const RopeArgs& a;
  const RopeLane& l;
  __device__ __forceinline__ RopePartners(const RopeArgs& args, const RopeLane& lane,
                                          const typename Raw<T, V>::type (&r)[U], char* lds)
      : p(rope_partner<V, WAY>(args, lane)), rows(reinterpret_cast<T*>(lds)), a(args), l(lane) {
    if constexpr (WAY != kRopeGather) return;
    wave_lds_fence();
    if (l.live) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        *reinterpret_cast<typename Raw<T, V>::type*>(
            reinterpret_cast<T*>(lds + u * kRopeRow) + l.sub * a.dim + l.at * V) = r[u];
    }
    wave_lds_fence();
  }
  __device__ __forceinline__ void get(const typename Raw<T, V>::type& r, int u,
                                      float (&o)[V]) const {
    if constexpr (WAY == kRopeGather) {
      const T* row = rows + u * (kRopeRow / sizeof(T)) + (l.live ? l.sub : 0) * a.dim;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = static_cast<float>(row[partner_of(a, l.at * V + i)]);
      return;
    }
    constexpr int N = V * sizeof(T) / 4;
    typename Raw<T, V>::type q;
    if constexpr (N == 1) {
      q = __builtin_bit_cast(
          typename Raw<T, V>::type,
          __builtin_amdgcn_ds_bpermute(4 * p.lane[0], __builtin_bit_cast(int, r)));
    } else {
      typedef int words __attribute__((ext_vector_type(N)));
      const words w = __builtin_bit_cast(words, r);
      words x;
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[i] = __builtin_amdgcn_ds_bpermute(
            4 * p.lane[i / (N / 2)], WAY == kRopeHalves && p.crossed ? w[(i + N / 2) % N] : w[i]);
      q = __builtin_bit_cast(typename Raw<T, V>::type, x);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = raw_at<T, V>(q, i);
  }
};

// One weight, widened (1 without weights).
template <typename T>
__device__ __forceinline__ float load_weight(const RopeArgs& a, const RopeSide& side, int i) {
  if (side.w == nullptr) return 1.0f;
  if (a.w_f32) {
    const float* w = static_cast<const float*>(side.w);
    return load_any<float, 1, false>(w + i, VBH_SPAN(w, a.dim));
  }
  const T* w = static_cast<const T*>(side.w);
  return static_cast<float>(load_any<T, 1, false>(w + i, VBH_SPAN(w, a.dim)));
}

template <typename W, int V>
__device__ __forceinline__ void widen_weights(const RopeArgs& a, const RopeSide& side,
                                              const RopeLane& l, float (&w)[V]) {
  const W* from = static_cast<const W*>(side.w);
  const typename Raw<W, V>::type r = load_any<W, V, false>(from + l.at * V, VBH_SPAN(from, a.dim));
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = raw_at<W, V>(r, i);
}
// The lane's V weights, widened (ones without weights).
template <typename T, int V>
__device__ __forceinline__ void load_weights(const RopeArgs& a, const RopeSide& side,
                                             const RopeLane& l, float (&w)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = 1.0f;
  if (side.w == nullptr) return;
  if (a.w_f32) widen_weights<float, V>(a, side, l, w);
  else widen_weights<T, V>(a, side, l, w);
}

// The weights of the partners of a lane's values (half pairing).
template <typename T, int V, int WAY>
__device__ __forceinline__ void partner_weights(const RopeArgs& a, const RopeSide& side,
                                                const RopeLane& l, const RopePartner<V>& p,
                                                const float (&w)[V], float (&o)[V]) {
  if constexpr (WAY == kRopeGather) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = load_weight<T>(a, side, partner_of(a, l.at * V + i));
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    o[i] = __int_as_float(__builtin_amdgcn_ds_bpermute(
        4 * p.lane[i / (V / 2)],
        __float_as_int(WAY == kRopeHalves && p.crossed ? w[(i + V / 2) % V] : w[i])));
}

// How a lane's V values turn: y_i = x_i c[i] + x_partner s[i], passing[i] where
// they do not (not with kRopeWhole).
template <int V>
struct Turn {
  float c[V], s[V];
  bool passing[V];
};

template <int V, bool ADJ, int WAY>
__device__ __forceinline__ void make_turn(const RopeArgs& a, const RopeLane& l,
                                          const float2* table, Turn<V>& t) {
  if constexpr (ADJ) {
    constexpr int N = V / 2;
    const int p0 = l.at * N;
    float c[N], si[N];
    // a run whose first pair passes reads another; n_freq may end inside a run, whose
    // rest lies in the table's last places, unwritten and unused
    read_turns<N>(table, WAY != kRopeWhole && p0 >= a.n_freq ? 0 : p0, c, si);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool pass = WAY != kRopeWhole && p0 + i >= a.n_freq;
      t.passing[2 * i] = t.passing[2 * i + 1] = pass;
      t.c[2 * i] = t.c[2 * i + 1] = pass ? 1.0f : c[i];
      t.s[2 * i] = pass ? 0.0f : -si[i];
      t.s[2 * i + 1] = pass ? 0.0f : si[i];
    }
  } else if constexpr (WAY == kRopeGather) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = l.at * V + i;
      const bool pass = e >= 2 * a.n_freq, first = e < a.n_freq;
      const float2 cs = table[table_place(pass ? 0 : first ? e : e - a.n_freq)];
      t.passing[i] = pass;
      t.c[i] = pass ? 1.0f : cs.x;
      t.s[i] = pass ? 0.0f : first ? -cs.y : cs.y;
    }
  } else {
    constexpr int H = WAY == kRopeWhole ? V : V / 2;  // values that turn alike
#pragma unroll
    for (int h = 0; h < V / H; ++h) {
      const int at = l.at * V + h * H;
      const bool pass = WAY != kRopeWhole && at >= 2 * a.n_freq, first = at < a.n_freq;
      float c[H], si[H];
      read_turns<H>(table, pass ? 0 : first ? at : at - a.n_freq, c, si);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        t.passing[h * H + i] = pass;
        t.c[h * H + i] = pass ? 1.0f : c[i];
        t.s[h * H + i] = pass ? 0.0f : first ? -si[i] : si[i];
      }
    }
  }
}

// N sums over aligned groups of 2^log2 lanes, step by step for all of them (the
// steps of wave_allreduce).
template <int N>
__device__ __forceinline__ void wave_sums(float (&v)[N], int log2) {
  if (log2 >= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0xB1>(v[i]);
  }
  if (log2 >= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0x4E>(v[i]);
  }
  if (log2 >= 3) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0x141>(v[i]);
  }
  if (log2 >= 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += dpp<0x140>(v[i]);
  }
  if (log2 >= 5) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]),
                                                      __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
  }
  if (log2 >= 6) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]),
                                                      __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
  }
}

// Sums of N values over the lanes of each vector, in every lane of it.  `scratch`:
// N * kRopeScratch floats of the wave's own, used where the lanes are no power of
// two: there each lane leaves its value and adds up its vector's.
template <int N>
__device__ __forceinline__ void vector_sums(const RopeArgs& a, const RopeLane& l, float (&v)[N],
                                            float* scratch) {
  if (a.tile.lanes_log2 >= 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = l.live ? v[i] : 0.0f;
    wave_sums<N>(v, a.tile.lanes_log2);
    return;
  }
  const int lanes = a.tile.lanes, line = (lanes + 3) & ~3;  // whole 16-byte reads
  wave_lds_fence();
  if (l.live) {
#pragma unroll
    for (int i = 0; i < N; ++i) scratch[i * kRopeScratch + l.sub * line + l.at] = v[i];
  }
  wave_lds_fence();
  const float* from = scratch + (l.live ? l.sub : 0) * line;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
  int j = 0;
  for (; j + 4 <= lanes; j += 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float4 q = *reinterpret_cast<const float4*>(from + i * kRopeScratch + j);
      v[i] += (q.x + q.y) + (q.z + q.w);
    }
  }
  const int rest = lanes - j;
  if (rest > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float4 q = *reinterpret_cast<const float4*>(from + i * kRopeScratch + j);
      v[i] += q.x + (rest > 1 ? q.y : 0.0f) + (rest > 2 ? q.z : 0.0f);
    }
  }
}

// One token's output vectors of one side, [heads, D] at `base`: stores through a
// buffer resource whose range check drops what lies behind them, so that lanes
// without a vector need no branch around the store (which would keep the compiler
// from overlapping the passes).  `base` is 16-byte aligned where V values are.
template <typename T, int V, int MEM>
struct RopeOut {
  __amdgpu_buffer_rsrc_t rsrc;
  T* base;
  Span span;
  __device__ __forceinline__ RopeOut(const RopeArgs& a, const RopeSide& side, int64_t token) {
    const int values = side.heads * a.dim;
    base = static_cast<T*>(side.y) + token * values;
    span = VBH_SPAN(static_cast<T*>(side.y), a.tokens * values);
    rsrc = __builtin_amdgcn_make_buffer_rsrc(
        base, static_cast<short>(0),
        __builtin_amdgcn_readfirstlane(values * static_cast<int>(sizeof(T))), kRawBufferWord3);
  }
  // Values `at` on, rounded to T; not `there`: dropped.
  __device__ __forceinline__ void store(int at, bool there, const float* o) const {
    if (!VBH_IN_SPAN(span, there ? base + at : base, V * sizeof(T))) return;
    typename Raw<T, V>::type r;
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = static_cast<T>(o[i]);
    const int off = there ? at * static_cast<int>(sizeof(T)) : INT_MAX;
    constexpr int N = V * sizeof(T) / 4;
    constexpr int kAux = MEM == kRopeStream ? kCacheNtSc1 : kCacheSc1;
    typedef int words __attribute__((ext_vector_type(N)));
    if constexpr (N == 4)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(words, r), rsrc, off, 0, kAux);
    else if constexpr (N == 2)
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(words, r), rsrc, off, 0, kAux);
    else
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, r), rsrc, off, 0, kAux);
  }
};

// Sum over a lane's values of x^2; 16-bit pairs on the dot-product unit.
template <typename T, int V>
__device__ __forceinline__ float squares(const typename Raw<T, V>::type& r) {
  float sum = 0.0f;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      typename Pair<T>::type p;
      p[0] = r[i];
      p[1] = r[i + 1];
      sum = Pair<T>::dot(p, p, sum);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fmaf(r[i], r[i], sum);
  }
  return sum;
}

// ---------------------------------------------------------------------------
// pair by pair
// ---------------------------------------------------------------------------

// A lane's k-th pair of a vector: its values' places, whether there are both, its
// number among the turning pairs or -1 where they pass.
struct RopePair {
  int a, b, p;
  bool has_a, has_b;
};
template <bool ADJ>
__device__ __forceinline__ RopePair rope_pair(const RopeArgs& a, const RopeLane& l, int k) {
  const int slots = (a.dim + 1) / 2, slot = l.at + k * kWave;
  const bool turns = slot < a.n_freq;
  RopePair r;
  r.p = turns ? slot : -1;
  if constexpr (ADJ) {
    r.a = 2 * slot;
    r.b = r.a + 1;
  } else {
    r.a = turns ? slot : a.n_freq + slot;
    r.b = r.a + (turns ? a.n_freq : slots - a.n_freq);
  }
  r.has_a = l.live && slot < slots;
  r.has_b = r.has_a && r.b < a.dim;
  return r;
}

template <typename T>
__device__ __forceinline__ float load_value(const T* x, bool there, const Span& s) {
  return there ? raw_at<T, 1>(load_any<T, 1>(x, s), 0) : 0.0f;
}

}  // namespace vbh
