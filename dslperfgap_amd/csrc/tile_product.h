// Matrix products on the matrix cores, tile by tile, for gfx950:
//
//   out[r, c] = sum over k of P[r, k] Q[c, k]
//
// A workgroup of WR x WC waves computes a tile of BR rows by BC columns; a wave holds
// RB x CB blocks of 16 x 16 fp32 sums.  k goes in stages of 128 bytes of each row or
// column (64 values of 16 bits, 32 of fp32), which the buffer loads write straight into
// the LDS, at least one stage ahead of the one that the matrix cores work on.
//
// An operand lies in memory with k contiguous ("rows": [r][k]) or with k the slow axis
// ("columns": [k][r]).  Columns of 16-bit values are turned on the way from the LDS to the
// registers (ds_read_b64_tr_b16).  Rows and values of k beyond the operand's end read as
// zeros: by the buffer resource's range, and within a row by an offset beyond it.  (Scalar offsets
// stay within the range too, `more`, which costs 0.5 to 1.8% of a backward call; behind a branch
// that only a tile's last stages take, 6%.)
//
// Bank conflicts: the LDS takes stages as the loads deliver them, 16 bytes per lane in
// lane order, so lanes ask for their 16-byte pieces in a permuted order instead (SQ counters
// show none for 16-bit operands; without it every second cycle of the reads is one):
//   rows: piece p of row r lies at p ^ (r / 2 % 8);
//   columns: piece p of line k lies at p ^ 4 (k % 4) ^ 2 (k / 8 % 2), of 32-bit values at
//   p ^ 4 (k / 4 % 2).
//
// MI355X, bf16, 256 x 256 tiles, us (TFLOP/s) beside the library's best kernel for the layout:
// 8192 x 8192 x 8192 deep, rows by rows 781 (1408; library 698, 1574), rows by columns
// 8192 x 4096 x 16384 823 (1335; 901, 1221), columns by columns 16384 x 4096 x 8192 808
// (1360; 1030, 1067).  Blocks of 32 x 32 reach 1280, 1170 and 1214 in the same scheme: their
// sums cross the registers twice as often per operation, and the card's power is the bound
// (the same loop without its loads runs at 1567, without its LDS reads at 1605, without
// either at 2120).  4 waves of 128 x 128: 1270.  Four buffers of half a stage: 1223 (rows of 64
// bytes), 1245 and 1270.
#pragma once

#include <type_traits>

#include "vbh_device.h"

namespace vbh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

template <typename T> struct Frag { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };

// acc[m][n] += sum over the fragments' k of a[m] b[n]: lane l holds row (column) l % 16 and
// the 16 bytes of k of quarter l / 16; of the sums column n = l % 16 and rows
// m = 4 (l / 16) + i.
__device__ __forceinline__ f32x4 multiply(const Frag<__bf16>::type& a, const Frag<__bf16>::type& b,
                                           const f32x4& acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(const Frag<_Float16>::type& a,
                                           const Frag<_Float16>::type& b, const f32x4& acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(const Frag<float>::type& a, const Frag<float>::type& b,
                                           f32x4 acc) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
  return acc;
}

constexpr int kStageBytes = 128;  // of k, per row
template <typename T> constexpr int kStageValues = kStageBytes / static_cast<int>(sizeof(T));
constexpr int kSteps = 2;         // fragments per stage
constexpr int kBlockRows = 16;    // of a fragment

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
  static_assert(kBytes % (16 * LANES) == 0 && LANES % kPieces == 0 &&
                    kLinesPerLoad % (COLUMNS && sizeof(T) == 4 ? 8 : 16) == 0,
                "whole loads, of lines whose permutation does not depend on the load");
  static_assert(!COLUMNS || kPieces >= 16, "room for the permutation");

  __amdgpu_buffer_rsrc_t rsrc;
  const T* base;     // of the resource: the next stage's first line
  int64_t line;      // bytes from one line to the next
  int64_t extent;    // bytes from base to the operand's end
  // Scalar offset of each load.  A lane's load is out of range where its own offset reaches the range
  // less this one, which therefore never passes the range.
  uint32_t more[kLoads];
  uint32_t offset;   // of the lane's first piece from base
  int k_left;        // rows: values of k that the lane's pieces have ahead of them
  Span span;

  // `from`: the tile's first line (columns: and first row) at k = 0; `lines`: lines from there on
  // that the operand has; `values`: values of a line from there on.
  __device__ __forceinline__ Operand(const T* from, int64_t ld, int64_t lines, int64_t values,
                                     const Span& s)
      : base(from), line(ld * static_cast<int64_t>(sizeof(T))), span(s) {
    const int t = static_cast<int>(threadIdx.x);
    const int at = t / kPieces, slot = t % kPieces;
    const int piece = !COLUMNS         ? slot ^ ((at >> 1) & 7)
                      : sizeof(T) == 2 ? slot ^ ((at & 3) << 2) ^ (((at >> 3) & 1) << 1)
                                       : slot ^ (at & 4);
    offset = static_cast<uint32_t>(at * line + piece * 16);
    extent = lines > 0 ? (lines - 1) * line + values * static_cast<int64_t>(sizeof(T)) : 0;
    k_left = static_cast<int>(values) - piece * (16 / static_cast<int>(sizeof(T)));
    range();
  }
  __device__ __forceinline__ void range() {
    const int bytes = __builtin_amdgcn_readfirstlane(
        static_cast<int>(extent < kMaxRange ? (extent > 0 ? extent : 0) : kMaxRange));
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      more[j] = min(static_cast<uint32_t>(j * kLinesPerLoad * line), static_cast<uint32_t>(bytes));
    rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), static_cast<short>(0),
                                             bytes, kRawBufferWord3);
  }
  // On (or back) by `stages`.
  __device__ __forceinline__ void move(int stages) {
    const int64_t by = stages * (COLUMNS ? kStageValues<T> * line : kStageBytes);
    base = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + by);
    extent -= by;
    k_left -= stages * kStageValues<T>;
    range();
  }

  // The next stage into `lds` (kBytes), and on to the one behind it.
  __device__ __forceinline__ void load(char* lds) {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    uint32_t from = offset;
    if constexpr (!COLUMNS) from = k_left > 0 ? offset : kNowhere;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      uint32_t at = from;
#ifdef VBH_DEBUG_BOUNDS
      const int64_t place = static_cast<int64_t>(from) + more[j];
      if (from != kNowhere && place < extent && place < kMaxRange &&
          !VBH_IN_SPAN(span, reinterpret_cast<const char*>(base) + place, 16))
        at = kNowhere;
#endif
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (lds_void*)(lds + (j * LANES + wave * kWave) * 16), 16, at, more[j], 0, 0);
    }
    move(1);
  }

  // The lane's fragment of the 16 rows of block `block` from row `base` (a multiple of 32) on at
  // step `step` of the stage in `lds`.
  __device__ static __forceinline__ typename Frag<T>::type fragment(const char* lds, int base,
                                                                    int block, int step) {
    const int row = base + block * kBlockRows;
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int quarter = lane >> 4;
    if constexpr (!COLUMNS) {
      // one address per step, blocks apart by an immediate offset
      const int from =
          (lane & 15) * kStageBytes + (((4 * step + quarter) ^ ((lane >> 1) & 7)) * 16);
      return *reinterpret_cast<const typename Frag<T>::type*>(lds + from + row * kStageBytes);
    } else if constexpr (sizeof(T) == 4) {
      // 16 lanes read 64 bytes of a line, the next ones as much 4 lines on
      typename Frag<T>::type f;
      const int from = quarter * 4 * kPieces * 16 + (lane & 15) * 4 +
                       (((block & 1) * 64) ^ ((quarter & 1) * 64)) + base * 4 + (block >> 1) * 128;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *reinterpret_cast<const float*>(lds + from + (16 * step + j) * kPieces * 16);
      return f;
    } else {
      // 16 lanes read 4 lines of 16 values and get one column of 4 each
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const int r = row + (lane & 3) * 4;  // of the lane's 8 bytes
      const int k = step * 32 + quarter * 8 + ((lane & 15) >> 2);
      const int piece = (r >> 3) ^ ((k & 3) << 2) ^ (((k >> 3) & 1) << 1);
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

// DEEP: four buffers of a whole stage instead of two, three stages ahead, for products of so few rows
// that their time is the read of Q.
template <typename T, int BR_, int BC_, int WR_, int WC_, bool P_COLUMNS, bool Q_COLUMNS,
          bool DEEP = false>
struct TileProduct {
  static constexpr int BR = BR_, BC = BC_, WR = WR_, WC = WC_;
  static constexpr int kLanes = WR * WC * kWave;
  static constexpr int RB = BR / WR / kBlockRows, CB = BC / WC / kBlockRows;  // blocks of a wave
  typedef Operand<T, BR, kLanes, P_COLUMNS> P;
  typedef Operand<T, BC, kLanes, Q_COLUMNS> Q;
  typedef typename Frag<T>::type F;
  // of the kernel's four buffers
  static constexpr int kPBuffer = DEEP ? P::kBytes + Q::kBytes : P::kBytes;
  static constexpr int kQBuffer = DEEP ? P::kBytes + Q::kBytes : Q::kBytes;

  f32x4 sums[RB][CB];

  __device__ static __forceinline__ int wave_row() {
    return (__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6) / WC) * (BR / WR);
  }
  __device__ static __forceinline__ int wave_col() {
    return (__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6) % WC) * (BC / WC);
  }

  // A stage's work in units: one fragment of Q against a step's RB fragments of P, RB matrix
  // instructions.  A fragment of Q is read kAhead units before its own, those of P all at once as
  // far ahead of their step.  The next stage's first ones are read behind the barrier, which
  // therefore stands kAhead units before the stage's end: by then nothing of this stage is left to
  // read, and its buffer takes the stage behind the next.  (kAhead 2, 3, 4 and 5 are within 1% of
  // each other; the loads ahead of the reads behind the barrier 1% slower.)
  static constexpr int kUnits = kSteps * CB, kAhead = CB > 3 ? 3 : CB, kBarrier = kUnits - kAhead;

  // Over k values of k.  The buffers are variables of their own, so that the compiler knows
  // which loads a read of the LDS has to wait for.
  // DEEP: stages are taken in a circle, from the part `from` / kFroms of them on: workgroups that
  // walk over equally aligned lines in step ask the same memory channels at a time (4 tokens by a
  // bf16 W of 32000 x 4096: 58.2 us, with each workgroup from a stage of its own 54.5; it makes no
  // difference to tiles that are bound by the matrix cores).
  static constexpr int kFroms = 64;
  __device__ __forceinline__ void run(P& p, Q& q, int64_t k, int from, char* p0, char* p1, char* q0,
                                      char* q1) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int c = 0; c < CB; ++c) sums[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int stages = static_cast<int>((k + kStageValues<T> - 1) / kStageValues<T>);
    const int wr = wave_row(), wc = wave_col();
    if constexpr (DEEP) {
      constexpr int kLoads = P::kLoads + Q::kLoads;
      const int first = static_cast<int>(static_cast<int64_t>(stages) * from / kFroms);
      int loaded = first;  // from the first stage on; past them all, zeros
      p.move(first);
      q.move(first);
      auto load = [&](char* to) {
        if (loaded == stages) {  // back to the first; behind the last again, past the end
          p.move(-stages);
          q.move(-stages);
        }
        if (loaded == stages + first) {
          p.move(stages);
          q.move(stages);
        }
        ++loaded;
        p.load(to);
        q.load(to + P::kBytes);
      };
      auto work = [&](char* at, char* before) {
        stage_barrier<2 * kLoads>();
        load(before);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          F a[RB], b[CB];
#pragma unroll
          for (int r = 0; r < RB; ++r) a[r] = P::fragment(at, wr, r, s);
#pragma unroll
          for (int c = 0; c < CB; ++c) b[c] = Q::fragment(at + P::kBytes, wc, c, s);
#pragma unroll
          for (int r = 0; r < RB; ++r) {
#pragma unroll
            for (int c = 0; c < CB; ++c) sums[r][c] = multiply(b[c], a[r], sums[r][c]);
          }
        }
      };
      load(p0);
      load(p1);
      load(q0);
      for (int s = 0; s < stages; s += 4) {
        work(p0, q1);
        work(p1, p0);
        work(q0, p1);
        work(q1, q0);
      }
      stage_barrier<0>();
      return;
    }
    F qf[kUnits], qn[kAhead], pf[kSteps][RB], pn[RB];
    auto unit_of = [&](const char* lds, int u) {
      return Q::fragment(lds, wc, u % CB, u / CB);
    };
    auto rows_of = [&](const char* lds, int step, F(&f)[RB]) {
#pragma unroll
      for (int r = 0; r < RB; ++r) f[r] = P::fragment(lds, wr, r, step);
    };
    // the stage in (pc, qc), then on to the one in (pn_, qn_)
    auto turn = [&](char* pc, char* qc, char* pn_, char* qn_) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (u == kBarrier) {
          stage_barrier<0>();
          rows_of(pn_, 0, pn);
          qn[0] = unit_of(qn_, 0);
          p.load(pc);
          q.load(qc);
        } else if (u < kBarrier) {
          qf[u + kAhead] = unit_of(qc, u + kAhead);
        } else {
          qn[u - kBarrier] = unit_of(qn_, u - kBarrier);
        }
        if (u % CB == CB - kAhead && u / CB + 1 < kSteps) rows_of(pc, u / CB + 1, pf[u / CB + 1]);
#pragma unroll
        for (int r = 0; r < RB; ++r)
          sums[r][u % CB] = multiply(qf[u], pf[u / CB][r], sums[r][u % CB]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) qf[u] = qn[u];
#pragma unroll
      for (int r = 0; r < RB; ++r) pf[0][r] = pn[r];
    };
    p.load(p0);
    q.load(q0);
    stage_barrier<0>();
    p.load(p1);
    q.load(q1);
    rows_of(p0, 0, pf[0]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) qf[u] = unit_of(q0, u);
    // two stages a turn: those behind the last read as zeros (a branch around one would give its
    // sums registers of their own, and spill)
    for (int s = 0; s < stages; s += 2) {
      turn(p0, q0, p1, q1);
      turn(p1, q1, p0, q0);
    }
    stage_barrier<0>();
  }

  // Calls f(row, column of the first of 4 consecutive columns, the 4 sums) for the lane's sums.
  template <typename F_>
  __device__ __forceinline__ void each(F_&& f) const {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int c = 0; c < CB; ++c)
        f(wave_row() + r * kBlockRows + (lane & 15),
          wave_col() + c * kBlockRows + 4 * (lane >> 4), sums[r][c]);
    }
  }
};

}  // namespace vbh
