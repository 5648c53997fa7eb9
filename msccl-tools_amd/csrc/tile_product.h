// A tile of a 16-bit matrix product on the matrix cores: out[r][l] = sum over k of L[l][k] R[r][k], sums in 32 bits.
//
// L runs along the output's rows (its contiguous dimension), R across them, so that the four registers of a
// 16 x 16 x 32 instruction's result are four neighbours of one output row.  Either operand may be stored with k
// contiguous ("row": one row of memory per l or r) or with k strided ("col": one row of memory per k).
//
// Data path: a workgroup copies the next 64 values of k of both operands from memory into LDS without passing through
// registers (16 bytes per lane), while its waves feed the matrix cores from the copy before.  The copies write LDS in lane order, so
// the bank swizzle is applied to the addresses they read from:
//   row operand: 128 bytes per row, the 16-byte unit u of row i sits at u ^ (i / 2 % 8): the sixteen rows that a
//                fragment read touches at one unit then cover all 64 banks;
//   col operand: one line of 2 * TILE bytes per k, 32-byte pair p of line k sits at p ^ (k % 4 + 4 * (k / 8 % 2)):
//                the transposing read takes 8 lines x 32 bytes per half wave, again all banks once.
// What lies outside an operand (rows behind the last, k behind the last) is asked for at an offset beyond the
// buffer resource's range: the hardware writes zeros for it and touches no memory.
#ifndef MSCCLX_TILE_PRODUCT_H
#define MSCCLX_TILE_PRODUCT_H

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mscclx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kStepK = 64;                      // values of k per step
constexpr unsigned kOutside = 0x80000000u;      // a byte offset that no operand holds
constexpr int kResourceBytes = 0x7ffffff0;      // range of the buffer resources: every valid offset is below, kOutside is not

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

// 16 bytes per lane from `resource` at `offset` (per lane) to LDS at m0 + 16 * lane.  Nothing else in these kernels uses m0.
__device__ __forceinline__ void copy_to_lds(unsigned lds, unsigned offset, i32x4 resource) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(resource) : "memory");
}
__device__ __forceinline__ i32x4 resource_at(const char* p) {
  const uint64_t a = (uint64_t)p;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), (int)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)), kResourceBytes, 0x00020000};
}

// The lanes' places in one operand's tile.  COL: k strided.  WAVES: waves of the workgroup.  CHUNKS copies make a step.
template <bool COL, int TILE, int WAVES>
struct Lanes {
  static constexpr int kBytes = TILE * kStepK * 2;
  static constexpr int kChunk = WAVES * 1024;
  static constexpr int kChunks = kBytes / kChunk;
  static constexpr int kUnitsPerLine = COL ? TILE / 8 : 8;       // 16-byte units of a line of LDS
  static constexpr int kLines = WAVES * 64 / kUnitsPerLine;      // lines per chunk
  static_assert(kChunks >= 1 && (COL ? TILE >= 128 : kLines % 16 == 0), "a copy covers whole swizzle patterns");
  unsigned offset[kChunks];
  int k[COL ? kChunks : 1];                                      // the lane's k (its first) in the step

  // `stride`: bytes between rows of memory; `valid`: rows (row) or columns (col) that exist
  __device__ __forceinline__ void place(int thread, int64_t stride, int valid) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int line = i * kLines + thread / kUnitsPerLine, unit = thread % kUnitsPerLine;
      if constexpr (COL) {
        const int from = (((unit >> 1) ^ ((line & 3) | ((line >> 3 & 1) << 2))) << 1) | (unit & 1);
        offset[i] = from * 8 < valid ? (unsigned)(line * stride) + from * 16 : kOutside;
        k[i] = line;
      } else {
        const int from = unit ^ (line >> 1 & 7);
        offset[i] = line < valid ? (unsigned)(line * stride) + from * 16 : kOutside;
        if (i == 0) k[0] = from * 8;   // a chunk is a multiple of 16 lines: the same for all
      }
    }
  }
  __device__ __forceinline__ void copy(unsigned lds, const char* from, int k_left) const {
    const i32x4 r = resource_at(from);
    if (k_left >= kStepK) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) copy_to_lds(lds + i * kChunk, offset[i], r);
    } else {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) copy_to_lds(lds + i * kChunk, k[COL ? i : 0] < k_left ? offset[i] : kOutside, r);
    }
  }
};

// Where an operand's steps begin.  k_left: values of k from there on.
struct RowSource {  // k contiguous
  const char* base;
  int64_t k;
  __device__ __forceinline__ const char* step(int s, int* k_left) {
    *k_left = (int)min((int64_t)kStepK, k - (int64_t)s * kStepK);
    return base + (int64_t)s * (kStepK * 2);
  }
};
struct ColSource {  // k strided
  const char* base;
  int64_t k, stride;
  __device__ __forceinline__ const char* step(int s, int* k_left) {
    *k_left = (int)min((int64_t)kStepK, k - (int64_t)s * kStepK);
    return base + (int64_t)s * kStepK * stride;
  }
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

  template <bool COL, int TILE, int F>
  static __device__ __forceinline__ void fragments(const char* lds, int first, int kk, int lane, i16x8 (&out)[F]) {
    if constexpr (COL) {
      const int k = kk * 32 + (lane >> 4) * 8 + (lane >> 2 & 3), swizzle = (lane >> 2 & 3) | ((lane >> 4 & 1) << 2);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const char* p = lds + k * (TILE * 2) + ((((first >> 4) + f) ^ swizzle) << 5) + (lane & 3) * 8;
        typedef __attribute__((address_space(3))) i16x4* lds_ptr;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * TILE * 2));
        out[f] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    } else {
      const int unit = (kk * 4 + (lane >> 4)) ^ (lane >> 1 & 7);
#pragma unroll
      for (int f = 0; f < F; ++f) out[f] = *(const i16x8*)(lds + (first + f * 16 + (lane & 15)) * 128 + unit * 16);
    }
  }

  // acc[l][r] += the product over all steps.  Every wave of the workgroup calls this with the same sources.
  template <class SL, class SR>
  static __device__ __forceinline__ void run(char* smem, int steps, const LLanes& ll, SL sl, const RLanes& rl, SR sr, f32x4 (&acc)[FL][FR]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l0 = wave % WL * (TL / WL), r0 = wave / WL * (TR / WR);
    typedef __attribute__((address_space(3))) char* lds_char;
    const unsigned lds = (unsigned)(uintptr_t)(lds_char)smem + wave * 1024;
    auto issue = [&](int s) {
      int k_left;
      const unsigned at = lds + s % STAGES * kStage;
      const char* p = sl.step(s, &k_left);
      ll.copy(at, p, k_left);
      p = sr.step(s, &k_left);
      rl.copy(at + LLanes::kBytes, p, k_left);
    };
    auto read = [&](int s, int kk, i16x8 (&a)[FL], i16x8 (&b)[FR]) {
      const char* at = smem + s % STAGES * kStage;
      fragments<RCOL, TR, FR>(at + LLanes::kBytes, r0, kk, lane, b);
      fragments<LCOL, TL, FL>(at, l0, kk, lane, a);
    };
    auto multiply = [&](const i16x8 (&a)[FL], const i16x8 (&b)[FR]) {
#pragma unroll
      for (int l = 0; l < FL; ++l)
#pragma unroll
        for (int r = 0; r < FR; ++r) acc[l][r] = Half<T>::mfma(a[l], b[r], acc[l][r]);
    };
    // a read from LDS, then a few products, and so on: neither waits for the other
    auto interleave = [&] {
      constexpr int kReads = FL * (LCOL ? 2 : 1) + FR * (RCOL ? 2 : 1), kEach = FL * FR / kReads > 0 ? FL * FR / kReads : 1;
#pragma unroll
      for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      }
      if constexpr (FL * FR > kReads * kEach) __builtin_amdgcn_sched_group_barrier(0x008, FL * FR - kReads * kEach, 0);
    };
    if (steps <= 0) return;
    i16x8 a0[FL], b0[FR], a1[FL], b1[FR];  // fragments of the step's first and second 32 values of k
    // Copies arrive in order: with the next STAGES - 2 steps' copies behind them, the awaited step's are there once no more are under way.
    // Where the last steps are not followed by others, everything is waited for.
    constexpr int kBehind = (STAGES - 2) * kCopies;
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
      if (s < steps) issue(s);
    if (steps >= STAGES) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kBehind + kCopies) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    read(0, 0, a0, b0);
    for (int s = 0; s < steps; ++s) {
      read(s, 1, a1, b1);
      multiply(a0, b0);
      interleave();
      // the copies of the next step have arrived, and every wave has read all of this one: its buffer takes the step STAGES further
      if (STAGES > 2 && s + STAGES <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kBehind) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (s + STAGES < steps) issue(s + STAGES);
      read(s + 1, 0, a0, b0);  // (behind the last step: what that buffer holds, for nothing)
      multiply(a1, b1);
      interleave();
    }
  }
};

}  // namespace mscclx
#endif
