// Matrix products on the matrix cores, tile by tile, for gfx950:
//
//   out[r, c] = sum over k of P[r, k] Q[c, k]
//
// A workgroup of WR x WC waves computes a tile of BR rows by BC columns; a wave holds
// RB x CB blocks of 32 x 32 fp32 sums.  k goes in stages of 128 bytes of each row or
// column (64 values of 16 bits, 32 of fp32), which the buffer loads write straight into
// the LDS, one stage ahead of the one that the matrix cores work on.
//
// An operand lies in memory with k contiguous ("rows": [r][k]) or with k the slow axis
// ("columns": [k][r]).  Columns of 16-bit values are turned on the way from the LDS to the
// registers (ds_read_b64_tr_b16).  Rows and values of k beyond the operand's end read as
// zeros: by the buffer resource's range, and within a row by an offset beyond it.
//
// Bank conflicts: the LDS takes stages as the loads deliver them, 16 bytes per lane in
// lane order, so lanes ask for their 16-byte pieces in a permuted order instead:
//   rows: piece p of row r lies at p ^ (r & 7);
//   columns: piece p of line k lies at p ^ 4 (k & 3), of 32-bit values at p ^ 2 (k & 4).
#pragma once

#include <type_traits>

#include "vbh_device.h"

namespace vbh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

template <typename T> struct Frag { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };

// acc[m][n] += sum over the fragments' k of a[m] b[n]: lane l holds row (column) l % 32 and
// the 16 bytes of k of half l / 32; of the sums column n = l % 32 and rows
// m = 8 (i / 4) + 4 (l / 32) + i % 4.
__device__ __forceinline__ f32x16 multiply(const Frag<__bf16>::type& a, const Frag<__bf16>::type& b,
                                           const f32x16& acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(const Frag<_Float16>::type& a,
                                           const Frag<_Float16>::type& b, const f32x16& acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(const Frag<float>::type& a, const Frag<float>::type& b,
                                           f32x16 acc) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
  return acc;
}

constexpr int kStageBytes = 128;  // of k, per row
template <typename T> constexpr int kStageValues = kStageBytes / static_cast<int>(sizeof(T));
constexpr int kSteps = 4;         // fragments per stage

// Beyond the range of every resource below.
constexpr uint32_t kNowhere = 0x7fffff00u;
constexpr int64_t kMaxRange = 0x40000000;

// One operand of a tile: `N` rows of the tile, in lines of `ld` values.
//   rows:    line r is row r, k runs along it
//   columns: line k holds the values of that k, rows run along it
template <typename T, int N, int LANES, bool COLUMNS>
struct Operand {
  static constexpr int kBytes = N * kStageBytes;           // of a stage
  static constexpr int kLoads = kBytes / 16 / LANES;       // of a lane per stage
  static constexpr int kPieces = COLUMNS ? N * static_cast<int>(sizeof(T)) / 16 : 8;  // of a line
  static constexpr int kLinesPerLoad = LANES / kPieces;
  static_assert(kBytes % (16 * LANES) == 0 && LANES % kPieces == 0 && kLinesPerLoad % 8 == 0,
                "whole loads, of lines whose permutation does not depend on the load");

  __amdgpu_buffer_rsrc_t rsrc;
  const T* base;     // of the resource
  int64_t line;      // bytes from one line to the next
  int64_t extent;    // bytes from base to the operand's end
  uint32_t offset;   // of the lane's first piece from the resource's base
  int k_left;        // rows: values of k that the lane's pieces have ahead of them
  Span span;

  // `base`: the tile's first line (columns: and first row) at k = 0; `lines`: lines from there on
  // that the operand has; `values`: values of a line from base on.
  __device__ __forceinline__ Operand(const T* from, int64_t ld, int64_t lines, int64_t values,
                                     const Span& s)
      : base(from), line(ld * static_cast<int64_t>(sizeof(T))), span(s) {
    const int t = static_cast<int>(threadIdx.x);
    const int at = t / kPieces, slot = t % kPieces;
    const int piece = !COLUMNS         ? slot ^ (at & 7)
                      : sizeof(T) == 2 ? slot ^ ((at & 3) << 2)
                                       : slot ^ ((at & 4) << 1);
    offset = static_cast<uint32_t>(at * line + piece * 16);
    extent = lines > 0 ? (lines - 1) * line + values * static_cast<int64_t>(sizeof(T)) : 0;
    k_left = static_cast<int>(values) - piece * (16 / static_cast<int>(sizeof(T)));
    range();
  }
  __device__ __forceinline__ void range() {
    const int64_t bytes = extent < kMaxRange ? (extent > 0 ? extent : 0) : kMaxRange;
    rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(base), static_cast<short>(0),
        __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), kRawBufferWord3);
  }

  // The next stage into `lds` (kBytes), and on to the one behind it.
  __device__ __forceinline__ void load(char* lds) {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    uint32_t from = offset;
    if constexpr (!COLUMNS) from = k_left > 0 ? offset : kNowhere;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const uint32_t more = static_cast<uint32_t>(j * kLinesPerLoad * line);
      uint32_t at = from;
#ifdef VBH_DEBUG_BOUNDS
      const int64_t place = static_cast<int64_t>(from) + more;
      if (from != kNowhere && place < extent && place < kMaxRange &&
          !VBH_IN_SPAN(span, reinterpret_cast<const char*>(base) + place, 16))
        at = kNowhere;
#endif
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (lds_void*)(lds + (j * LANES + wave * kWave) * 16), 16, at, more, 0, 0);
    }
    const int64_t step = COLUMNS ? kStageValues<T> * line : kStageBytes;
    base = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + step);
    extent -= step;
    k_left -= kStageValues<T>;
    range();
  }

  // The lane's fragment of rows `row` .. `row` + 31 at step `step` of the stage in `lds`.
  __device__ static __forceinline__ typename Frag<T>::type fragment(const char* lds, int row,
                                                                    int step) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int half = lane >> 5;
    if constexpr (!COLUMNS) {
      // row is a multiple of 32: one address per step, blocks apart by an immediate offset
      const int from = (lane & 31) * kStageBytes + (((2 * step + half) ^ (lane & 7)) * 16);
      return *reinterpret_cast<const typename Frag<T>::type*>(lds + from + row * kStageBytes);
    } else if constexpr (sizeof(T) == 4) {
      // 32 lanes read 128 bytes of a line, the others as much 4 lines on
      typename Frag<T>::type f;
      const int from = half * 4 * kPieces * 16 + (lane & 31) * 4 + ((row * 4) ^ (half * 128));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *reinterpret_cast<const float*>(lds + from + (8 * step + j) * kPieces * 16);
      return f;
    } else {
      // 16 lanes read 4 lines of 16 values and get one column of 4 each
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const int r = row + (lane & 16) + (lane & 3) * 4;  // of the lane's 8 bytes
      const int k = step * 16 + half * 8 + ((lane & 15) >> 2);
      const int piece = (r >> 3) ^ ((k & 3) << 2);
      const char* from = lds + (k * kPieces + piece) * 16 + (r & 7) * 2;
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(from));
      const s16x4 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(from + 4 * kPieces * 16));
      const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(typename Frag<T>::type, both);
    }
  }
};

// Every stage that this wave has asked for is in the LDS but the last `PENDING` loads, and every
// wave of the workgroup is past its last reads.
template <int PENDING>
__device__ __forceinline__ void stage_barrier() {
  static_assert(PENDING >= 0 && PENDING < 64, "six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory");
}

template <typename T, int BR_, int BC_, int WR_, int WC_, bool P_COLUMNS, bool Q_COLUMNS>
struct TileProduct {
  static constexpr int BR = BR_, BC = BC_, WR = WR_, WC = WC_;
  static constexpr int kLanes = WR * WC * kWave;
  static constexpr int RB = BR / WR / 32, CB = BC / WC / 32;  // blocks of a wave
  typedef Operand<T, BR, kLanes, P_COLUMNS> P;
  typedef Operand<T, BC, kLanes, Q_COLUMNS> Q;
  static constexpr int kLdsBytes = 2 * (P::kBytes + Q::kBytes);

  f32x16 sums[RB][CB];

  __device__ static __forceinline__ int wave_row() {
    return (__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6) / WC) * (BR / WR);
  }
  __device__ static __forceinline__ int wave_col() {
    return (__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6) % WC) * (BC / WC);
  }

  __device__ __forceinline__ void stage(const char* p, const char* q) {
    const int r0 = wave_row(), c0 = wave_col();
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      typename Frag<T>::type pf[RB], qf[CB];
#pragma unroll
      for (int r = 0; r < RB; ++r) pf[r] = P::fragment(p, r0 + r * 32, s);
#pragma unroll
      for (int c = 0; c < CB; ++c) qf[c] = Q::fragment(q, c0 + c * 32, s);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
#pragma unroll
        for (int c = 0; c < CB; ++c) sums[r][c] = multiply(qf[c], pf[r], sums[r][c]);
      }
    }
  }

  // Over k values of k.  The four buffers are variables of their own, so that the compiler knows
  // which loads a read of the LDS has to wait for.
  __device__ __forceinline__ void run(P& p, Q& q, int64_t k, char* p0, char* p1, char* q0,
                                      char* q1) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int c = 0; c < CB; ++c) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[r][c][i] = 0.0f;
      }
    }
    const int stages = static_cast<int>((k + kStageValues<T> - 1) / kStageValues<T>);
    p.load(p0);
    q.load(q0);
    // two stages a turn: one behind the last reads as zeros (a branch around it would give its
    // sums registers of their own, and spill)
    for (int s = 0; s < stages; s += 2) {
      stage_barrier<0>();
      p.load(p1);
      q.load(q1);
      stage(p0, q0);
      stage_barrier<0>();
      p.load(p0);
      q.load(q0);
      stage(p1, q1);
    }
    stage_barrier<0>();
  }

  // Calls f(row, column of the first of 4 consecutive columns, block row, block column, quarter)
  // for each group of sums that lie in consecutive columns: values 4 quarter .. + 3 of the block.
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int c = 0; c < CB; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f(wave_row() + r * 32 + (lane & 31), wave_col() + c * 32 + 8 * i + 4 * (lane >> 5), r, c, i);
      }
    }
  }
};

}  // namespace vbh
