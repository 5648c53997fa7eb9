// A tile of a 16-bit matrix product on the matrix cores: out[r][l] = sum over k of L[l][k] R[r][k], sums in 32 bits.
//
// L runs along the output's rows (its contiguous dimension), R across them, so that four registers of a
// matrix instruction's result are four neighbours of one output row.  Either operand may be stored with k
// contiguous ("row": one row of memory per l or r) or with k strided ("col": one row of memory per k).
//
// Data path: a workgroup copies the next 64 values of k of both operands from memory into LDS without passing through
// registers (16 bytes per lane), while its waves feed the matrix cores from the copy before.  The copies write LDS in
// lane order, so the bank swizzle is applied to the addresses they read from:
//   row operand: 128 bytes per row, the 16-byte unit u of row i sits at u ^ (i / 2 % 8): the sixteen rows that a
//                fragment read touches at one unit then cover all 64 banks;
//   col operand: one line of 2 * TILE bytes per k, 32-byte pair p of line k sits at p ^ swizzle_of(k): the transposing
//                read takes 8 lines x 1 pair per half wave, again all banks once.
// What lies outside an operand (rows behind the last, k behind the last) is asked for at an offset beyond the
// buffer resource's range: the hardware writes zeros for it and touches no memory.
#ifndef MSCCLX_TILE_PRODUCT_H
#define MSCCLX_TILE_PRODUCT_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "step_walk.h"

namespace mscclx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kStepK = 64;                      // values of k per step
constexpr unsigned kOutside = 0x80000000u;      // a byte offset that no operand holds
constexpr int kResourceBytes = 0x7ffffff0;      // range of the buffer resources: every valid offset is below, kOutside is not
constexpr int kUnitRows = 64;                   // rows that have one base address, where a row operand's rows have several

template <class T> struct Half;
template <> struct Half<__bf16> {
  typedef bf16x4 x4;
  typedef bf16x8 x8;
  static __device__ __forceinline__ f32x4 mfma(i16x8 a, i16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Half<_Float16> {
  typedef f16x4 x4;
  typedef f16x8 x8;
  static __device__ __forceinline__ f32x4 mfma(i16x8 a, i16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// 16 bytes per lane from `resource` at `offset` (per lane) + `further` to LDS at m0 + 16 * lane.  Nothing else in these
// kernels uses m0.  A vector instruction may have written `resource` just before (resource_at): a load wants five wait
// states behind it, which the compiler does not see to in here.
__device__ __forceinline__ void copy_to_lds(unsigned lds, unsigned offset, i32x4 resource, int further) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(offset), "s"(resource), "s"(further) : "memory");
}
__device__ __forceinline__ i32x4 resource_at(const char* p) {
  const uint64_t a = (uint64_t)p;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), (int)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)), kResourceBytes, 0x00020000};
}

__device__ __forceinline__ int swizzle_of(int k) { return (k & 3) | ((k >> 3 & 1) << 2); }

// The lanes' places in one operand's tile.  COL: k strided.  WAVES: waves of the workgroup.  CHUNKS copies make a step.
template <bool COL, int TILE, int WAVES>
struct Lanes {
  static constexpr int kBytes = TILE * kStepK * 2;
  static constexpr int kChunk = WAVES * 1024;
  static constexpr int kChunks = kBytes / kChunk;
  static constexpr int kUnitsPerLine = COL ? TILE / 8 : 8;       // 16-byte units of a line of LDS
  static constexpr int kLines = WAVES * 64 / kUnitsPerLine;      // lines per chunk
  static_assert(kChunks >= 1 && (COL ? TILE >= 128 : kLines % 16 == 0 && kUnitRows % kLines == 0), "a copy covers whole swizzle patterns");
  unsigned offset[kChunks];
  int k[COL ? kChunks : 1];                                      // the lane's k (its first) in the step

  // `stride`: bytes between rows of memory; `valid(unit)`: rows of the unit (row, counted from its base) or columns
  // (col) that exist.  A col operand's rows repeat themselves within a step with `period`, if it is less than a step.
  template <class F> __device__ __forceinline__ void place(int thread, int64_t stride, F valid, int period = kStepK) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      int line = i * kLines + thread / kUnitsPerLine;
      const int unit = thread % kUnitsPerLine;
      if constexpr (COL) {
        const int from = (((unit >> 1) ^ swizzle_of(line)) << 1) | (unit & 1);
        k[i] = line & (period - 1);
        offset[i] = from * 8 < valid(0) ? (unsigned)(k[i] * stride) + from * 16 : kOutside;
      } else {
        const int from = unit ^ (line >> 1 & 7);
        if (i == 0) k[0] = from * 8;   // a chunk is a multiple of 16 lines: the same for all
        line %= kUnitRows;
        offset[i] = line < valid(i * kLines / kUnitRows) ? (unsigned)(line * stride) + from * 16 : kOutside;
      }
    }
  }
  // copy `i` of a step that has `k_left` values of k
  __device__ __forceinline__ void copy(int i, unsigned lds, i32x4 from, int further, int k_left) const {
    copy_to_lds(lds + i * kChunk, k[COL ? i : 0] < k_left ? offset[i] : kOutside, from, further);
  }
};

// Where an operand's copies read: `base(i)`, the resource of the rows of unit i (row) or of all (col), for step after
// step `next()`; then `further` is what they add to it, and `left` the values of k from the step's first on.  Behind
// the last step nothing is left.
template <int TILE> struct RowSource : StepWalk<kStepK, 2 * kStepK> {  // k contiguous
  static constexpr int kUnits = (TILE + kUnitRows - 1) / kUnitRows;
  i32x4 bases[kUnits];
  // at(i): the address of unit i's first row.  first: the step to begin with; those in front of it come last
  template <class F> __device__ __forceinline__ RowSource(F at, int k, int first = 0) : StepWalk(k, first) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) bases[i] = resource_at(at(i));
  }
  __device__ __forceinline__ i32x4 base(int i) const { return bases[i]; }
};
struct ColSource {  // k strided
  static constexpr int further = 0;
  const char* at;
  int64_t stride;
  int left, k, turn;
  // again: the rows are gone through a second time, behind whole steps
  __device__ __forceinline__ ColSource(const char* at, int k, int64_t stride, bool again = false)
      : at(at - kStepK * stride), stride(stride), left(k + kStepK), k(k), turn(again ? (k + kStepK - 1) / kStepK : -1) {}
  __device__ __forceinline__ void next() {
    at += kStepK * stride, left -= kStepK;
    if (turn-- == 0) {
      const int rows = (k + kStepK - 1) / kStepK * kStepK;
      at -= rows * stride, left += rows;
    }
  }
  __device__ __forceinline__ i32x4 base(int) const { return resource_at(at); }
};

// TL x TR: the workgroup's tile, cut among WL x WR waves; STAGES: steps held in LDS, a power of two.
template <class T, int TL, int TR, int WL, int WR, int STAGES, bool LCOL, bool RCOL>
struct TileProduct {
  static constexpr int kWaves = WL * WR, kThreads = kWaves * 64;
  static constexpr int FL = TL / WL / 16, FR = TR / WR / 16;  // fragments of a wave
  typedef Lanes<LCOL, TL, kWaves> LLanes;
  typedef Lanes<RCOL, TR, kWaves> RLanes;
  static constexpr int kStage = LLanes::kBytes + RLanes::kBytes;
  static constexpr int kLdsBytes = STAGES * kStage;
  static constexpr int kCopies = LLanes::kChunks + RLanes::kChunks;  // of a wave, per step

  // where in the tile a lane's results of fragment f lie: l of the first of its four neighbours, and r
  static __device__ __forceinline__ int l_of(int thread, int f) { return (thread >> 6) % WL * (TL / WL) + f * 16 + (thread >> 4 & 3) * 4; }
  static __device__ __forceinline__ int r_of(int thread, int f) { return (thread >> 6) / WL * (TR / WR) + f * 16 + (thread & 15); }

  // Stores want 16 bytes per lane.  A lane holds four neighbours of fragment f and four of f + 1; lanes 16 apart swap
  // one of them, so that each has eight neighbours of one fragment: 64 bytes of an output row per store.  -> their
  // place in the tile, l
  static __device__ __forceinline__ int l_of_pair(int thread, int f) {
    const int group = thread >> 4 & 3;
    return (thread >> 6) % WL * (TL / WL) + (f + (group & 1)) * 16 + (group >> 1) * 8;
  }
  template <class X4> static __device__ __forceinline__ u32x4 pair_up(X4 first, X4 second) {
    const u32x2 a = __builtin_bit_cast(u32x2, first), b = __builtin_bit_cast(u32x2, second);
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false));
    return u32x4{x[0], y[0], x[1], y[1]};
  }

  // fragment f of a step's half
  template <bool COL, int TILE>
  static __device__ __forceinline__ i16x8 fragment(const char* lds, int first, int half, int lane, int f) {
    const int group = lane >> 4;  // of eight values of k
    if constexpr (COL) {
      typedef __attribute__((address_space(3))) i16x4* lds_ptr;
      const int within = group * 8 + (lane >> 2 & 3);  // (half a step further the swizzle is the same)
      const char* p = lds + (half * 32 + within) * (TILE * 2) + ((((first >> 4) + f) ^ swizzle_of(within)) << 5) + (lane & 3) * 8;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * TILE * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *(const i16x8*)(lds + (first + f * 16 + (lane & 15)) * 128 + ((half * 4 + group) ^ (lane >> 1 & 7)) * 16);
    }
  }

  // acc[l][r] += the product over all steps.  Every wave of the workgroup calls this with the same sources.
  template <class SL, class SR>
  static __device__ __forceinline__ void run(char* smem, int steps, const LLanes& ll, SL sl, const RLanes& rl, SR sr, f32x4 (&acc)[FL][FR]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l0 = wave % WL * (TL / WL), r0 = wave / WL * (TR / WR);
    typedef __attribute__((address_space(3))) char* lds_char;
    const unsigned lds = (unsigned)(uintptr_t)(lds_char)smem + wave * 1024;
    auto copy = [&](int s, int i) {
      const unsigned at = lds + s % STAGES * kStage;
      if (i < LLanes::kChunks) ll.copy(i, at, sl.base(LCOL ? 0 : i * LLanes::kLines / kUnitRows), sl.further, sl.left);
      else i -= LLanes::kChunks, rl.copy(i, at + LLanes::kBytes, sr.base(RCOL ? 0 : i * RLanes::kLines / kUnitRows), sr.further, sr.left);
    };
    struct Fragments {  // of half a step
      i16x8 a[FL], b[FR];
    };
    constexpr int kUnits = FL + FR;
    auto read = [&](Fragments& f, int s, int half, int u) {  // unit u: all of r, then of l, as the products want them
      const char* at = smem + s % STAGES * kStage;
      if (u < FR) f.b[u] = fragment<RCOL, TR>(at + LLanes::kBytes, r0, half, lane, u);
      else f.a[u - FR] = fragment<LCOL, TL>(at, l0, half, lane, u - FR);
    };
    // One fragment row of products after another; between them the next half's reads and, in the second half, the
    // copies, so that neither LDS nor the path to it gets all of a step's requests at once.
    auto multiply = [&](const Fragments& f, int l) {
#pragma unroll
      for (int r = 0; r < FR; ++r) acc[l][r] = Half<T>::mfma(f.a[l], f.b[r], acc[l][r]);
    };
    if constexpr (STAGES == 1) {  // nothing is read ahead: other workgroups of the compute unit fill the time
      for (int s = 0; s < steps; ++s) {
        sl.next(), sr.next();
#pragma unroll
        for (int i = 0; i < kCopies; ++i) copy(0, i);
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          Fragments f;
#pragma unroll
          for (int u = 0; u < kUnits; ++u) read(f, 0, half, u);
#pragma unroll
          for (int l = 0; l < FL; ++l) multiply(f, l);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      return;
    }
    Fragments now, next;
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      sl.next(), sr.next();
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy(s, i);
    }
    // copies arrive in order: the awaited step's are there once only those of the steps behind it are under way
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * kCopies) : "memory");
#pragma unroll
    for (int u = 0; u < kUnits; ++u) read(now, 0, 0, u);
    // Where registers are left, sums of four steps are added up, not one step to the sum of all before it: with few
    // tokens one of them can make the whole loss, and its logit's rounding errors a large part of it.
    constexpr bool kInTwo = STAGES > 2;
    f32x4 total[kInTwo ? FL : 1][kInTwo ? FR : 1] = {};
    auto add_up = [&] {
#pragma unroll
      for (int l = 0; l < FL; ++l)
#pragma unroll
        for (int r = 0; r < FR; ++r) total[l][r] += acc[l][r], acc[l][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    for (int s = 0; s < steps; ++s) {
      if constexpr (kInTwo)
        if (s % 4 == 0) add_up();
#pragma unroll
      for (int l = 0; l < FL; ++l) {
#pragma unroll
        for (int u = l * kUnits / FL; u < (l + 1) * kUnits / FL; ++u) read(next, s, 1, u);
        multiply(now, l);
        __builtin_amdgcn_sched_barrier(0);
      }
      // the copies of the next step have arrived, and every wave has read all of this one: its buffer takes the step
      // STAGES further
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * kCopies) : "memory");
      sl.next(), sr.next();
#pragma unroll
      for (int l = 0; l < FL; ++l) {
#pragma unroll
        for (int i = l * kCopies / FL; i < (l + 1) * kCopies / FL; ++i) copy(s + STAGES, i);
#pragma unroll
        for (int u = l * kUnits / FL; u < (l + 1) * kUnits / FL; ++u) read(now, s + 1, 0, u);  // (behind the last step: for nothing)
        multiply(next, l);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup
    if constexpr (kInTwo) {
      add_up();
#pragma unroll
      for (int l = 0; l < FL; ++l)
#pragma unroll
        for (int r = 0; r < FR; ++r) acc[l][r] = total[l][r];
    }
  }
};

}  // namespace mscclx
#endif
