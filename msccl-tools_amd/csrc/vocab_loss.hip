// Softmax cross entropy over a vocabulary that is cut into the ranks' pieces, with its gradients, without keeping the
// logits.
//
//   z[n][v]  = sum over d of x[n][d] w[v][d]        w: the ranks' rows one under the other
//   lse[n]   = log sum over v of exp z[n][v],   loss[n] = lse[n] - z[n][label[n]]
//   G[n][v]  = g[n] (exp(z[n][v] - lse[n]) - [v = label[n]]),   dx = G w,   dw = transposed(G) x
//
// Tokens go through in pieces of at most `piece` rows; per piece, three products on the matrix cores (tile_product.h):
//   logits   z of a tile of vocabulary x tokens stays in registers; what leaves are, for each token and each wave's part of the
//            vocabulary, the maximum m (in units of log 2) and the sum of exp(z - m), and with gradients E = exp(z - m) in 16 bits;
//   tokens   a token's (m, sum) become its lse and loss, and its E becomes G in place: G = (E exp(m - lse) - [label]) g / max|g|;
//   dx, dw   the two products, on G.  dx sums over the whole vocabulary: where its tiles do not fill the chip, that
//            axis is cut and the parts are added by workgroups that dw's launch has more.
// Tokens whose label is ignored have rows of zeros in G.  With more than kWideTokens tokens they are left out: G, and a
// copy of x beside it, hold the others' rows one behind the other, so that they cost nothing in the two products (of
// 8192 tokens x 131072 x 4096 with 15 % ignored: 20.4 -> 18.9 ms).  Their x is never read for a gradient: the copy has
// zeros there, or nothing.
// With few tokens, up to kWideTokens if they are few for each rank, memory and not the matrix cores sets the time, and
// nothing is lost to 16 bits on the way: the logits are kept in 32 bits instead of E, and G is kept as two 16-bit
// numbers, itself rounded and what that left (16 bits of it in bf16, 22 in fp16).  The products take the second ones as
// more rows.  (With so few tokens single values of G decide about a rank's dw, and some ranks hold no label: rounded
// once, dw was up to 1.9 times as far off as with G in 32 bits.)  With more tokens E and G are both rounded, each
// relative to its own size (bf16 2^-8, fp16 2^-11 at the most), with 2^15 as unit in fp16, so that probabilities down
// to 2^-29 are normal numbers; |g| is divided by its largest value for the same reason and multiplied back in 32 bits
// behind the products.  In fp16 a token's G is therefore off by up to 2^-40 of the largest |g| in each of the two roundings,
// whatever its own g: over 32000 rows at most 2^-24 of it times the largest |w| in the token's dx, which with both up to 1 is one
// step of the smallest numbers that dx holds.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>
#include <type_traits>
#include <vector>

#include "plan.h"
#include "tile_product.h"

namespace mscclx {
namespace {

constexpr int kMaxRanks = MSCCLX_VOCAB_LOSS_MAX_RANKS;
constexpr int kComputeUnits = 256;
constexpr int kTile = 256;              // columns of G are padded to a multiple of it
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 1.0 / (double)kLog2e;  // what takes the rounded kLog2e back

// The ranks' pieces of the vocabulary, passed to the kernels by value.  Units of kUnitRows rows; none spans two ranks,
// a tile may.  What pads a rank's last unit, or the last tile, counts as outside.
struct Pieces {
  int ranks, tiles;
  int rows[kMaxRanks];
  int unit0[kMaxRanks + 1];  // the rank's first unit
  int first[kMaxRanks + 1];  // the rank's first row in the whole vocabulary
  const char* w[kMaxRanks];
  __host__ __device__ int64_t columns() const { return (int64_t)tiles * kTile; }  // of E and G
  // Rows of a multiple of 2^16 columns would meet in one of memory's channels: they lie a cache line further apart (dx of
  // 2048 x 65536 x 1024: 251 us, without 280; 4096 x 65536 x 2048 837 / 852; with 32768 rows no shorter).
  __host__ __device__ int64_t stride() const { return columns() + (columns() % 65536 == 0 ? 64 : 0); }
};

// Which rank holds something: the ranks' ends, one in each lane, are compared at once.  (A loop over the ranks waits
// for memory at every turn.)
struct Ends {
  int end, ranks;
  __device__ __forceinline__ Ends(const int* ends, int ranks) : ranks(ranks) {
    const int lane = threadIdx.x & 63;
    end = lane < ranks ? ends[lane] : 0x7fffffff;
  }
  __device__ __forceinline__ int rank_of(int at) const { return min((int)__popcll(__ballot(at >= end)), ranks - 1); }
};

// Unit `unit` of the padded vocabulary
struct Unit {
  int rank, row;  // its rank, and its first row there
  int rows;       // from that row on; may be none, or less
  __device__ __forceinline__ Unit(const Pieces& p, const Ends& ends, int unit) : rank(__builtin_amdgcn_readfirstlane(ends.rank_of(unit))) {
    row = (unit - p.unit0[rank]) * kUnitRows;
    rows = p.rows[rank] - row;
  }
};

struct Grads {
  char* dw[kMaxRanks];
};

struct Labels {
  const void* at;
  int wide;  // 64-bit
  long long ignore;
  int64_t vocab;
  // -1: ignored, -2: no label of the vocabulary
  __device__ __forceinline__ int get(int64_t n) const {
    const long long v = wide ? ((const long long*)at)[n] : (long long)((const int*)at)[n];
    return v == ignore ? -1 : v < 0 || v >= vocab ? -2 : (int)v;
  }
};

// A token's g / max |g|: kept in `factor` where every token has its own, else the sign of the one number.
struct Upstream {
  const float* at;
  const float* factor;  // null: one number for all
  __device__ __forceinline__ float get(int64_t n, int label) const {
    if (factor) return factor[n];
    const float g = *at;
    return label == -1 ? 0.f : label < 0 ? NAN : g == 0.f ? 0.f : g / fabsf(g);
  }
};

// Exponents are kept in units of log 2: exp(z - m) = exp2(z log2(e) - M) with M = m log2(e), one multiply-add and one
// instruction.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
template <class T> constexpr float kUnit = std::is_same_v<T, _Float16> ? 32768.0f : 1.0f;

// How a workgroup's tile is cut.  Large: one workgroup of eight waves per compute unit.  Middle: two of four waves, for
// products whose large tiles would not fill the chip.  Small: three, for those whose middle ones would not.  Thin: four
// of four waves, each one step at a time, for products that write more than they read.  Few: at most 32 tokens, with
// four steps of copies under way, because then memory is all that counts.
template <int L, int R, int WL, int WR, int STAGES, int WAVES> struct Shape {  // WAVES: per SIMD, at least
  static constexpr int kL = L, kR = R, kWavesL = WL, kWavesR = WR, kThreads = WL * WR * 64, kWaves = WAVES;
  template <class T, bool LCOL, bool RCOL> using Product = TileProduct<T, L, R, WL, WR, STAGES, LCOL, RCOL>;
};
typedef Shape<256, 256, 2, 4, 2, 2> Large;
// dx's l is W^T, whose fragments take two reads of shared memory and r's one: with 4 x 2 waves each takes half as many
// of them.  At 8192 tokens of 4096 and 32768 rows dx takes 1547 us, with 2 x 4 waves 1577.
typedef Shape<256, 256, 4, 2, 2, 2> LargeDx;
typedef Shape<128, 128, 2, 2, 2, 2> Middle;
typedef Shape<128, 64, 2, 2, 2, 3> Small;
typedef Shape<128, 128, 2, 2, 1, 4> Thin;
typedef Shape<128, 32, 4, 1, 4, 2> Few;

enum { kStats = 0, kKeep = 1, kGradient = 2, kLogits = 3 };
constexpr int kWideTokens = 128;  // up to so many the logits are kept in 32 bits and G twice

struct LogitsArgs {
  const char* x;
  int64_t x_stride;  // bytes
  int64_t w_stride;
  int hidden, tokens, token_tiles;
  int apart;         // so many tiles of the vocabulary begin at the same k; 0: all
  int64_t token0;    // of the labels, lse and factors
  Labels labels;
  Upstream upstream;
  const int* pos;    // a token's row of E or G, -1: none; null: its own
  float2* stats;     // [tokens][waves' parts of the vocabulary]
  float* z_label;
  void* e;           // [rows][stride]: E or G, or with kLogits the logits in 32 bits
  const float* lse;
};

// Tiles in an order that keeps the workgroups of one XCD (every eighth of the grid) on neighbouring tiles: columns of
// up to kBand row tiles share what they read.  Of 8, 4 and 2, at 8192 tokens of 4096 and 32768 rows: logits kept 1697,
// 1651 and 1690 us, not kept 1522, 1511 and 1571; dx 1597, 1577 and 1578; dw 1622, 1607 and 1632.
constexpr int kBand = 4;
__device__ __forceinline__ int xcd_order(int id, int total) {
  const int per = total / 8;
  return id < per * 8 ? id % 8 * per + id / 8 : id;
}
__device__ __forceinline__ void tile_in_band(int id, int rows, int cols, int* row, int* col) {
  const int band = kBand * cols, at = id / band * kBand, high = min(kBand, rows - at), in = id % band;
  *row = at + in % high;
  *col = in / high;
}
__device__ __forceinline__ void tile_of(int id, int rows, int cols, int* row, int* col) { tile_in_band(xcd_order(id, rows * cols), rows, cols, row, col); }

template <class T, int MODE, class Shape>
__global__ void __launch_bounds__(Shape::kThreads, Shape::kWaves) logits_kernel(const Pieces pieces, const LogitsArgs a) {
  typedef typename Shape::template Product<T, false, false> Product;
  constexpr int TL = Shape::kL, TR = Shape::kR, kPart = TL / Shape::kWavesL;  // vocabulary of a wave
  __shared__ __attribute__((aligned(1024))) char smem[Product::kLdsBytes];
  const Ends ends(pieces.unit0 + 1, pieces.ranks);
  int tt, at;
  tile_of(blockIdx.x, a.token_tiles, pieces.tiles * (kTile / TL), &tt, &at);
  const int n0 = tt * TR, tokens = min(TR, a.tokens - n0);
  f32x4 acc[Product::FL][Product::FR] = {};
  {
    const int steps = (a.hidden + kStepK - 1) / kStepK, first = a.apart ? at / a.apart % steps : 0;
    typename Product::LLanes ll;
    typename Product::RLanes rl;
    ll.place(threadIdx.x, a.w_stride, [&](int i) { return Unit(pieces, ends, at * (TL / kUnitRows) + i).rows; });
    rl.place(threadIdx.x, a.x_stride, [&](int i) { return tokens - i * kUnitRows; });
    Product::run(smem, steps, ll,
                 RowSource<TL>([&](int i) {
                   const Unit u(pieces, ends, at * (TL / kUnitRows) + i);
                   return pieces.w[u.rank] + u.row * a.w_stride;
                 }, a.hidden, first),
                 rl, RowSource<TR>([&](int i) { return a.x + (n0 + i * kUnitRows) * a.x_stride; }, a.hidden, first), acc);
  }
  const int64_t ld = pieces.stride();
  const int lane = threadIdx.x & 63, part = (threadIdx.x >> 6) % Shape::kWavesL;
  // the wave's part of the vocabulary: whole units, or part of one
  constexpr int kOfWave = kPart < kUnitRows ? kPart : kUnitRows, kWaveUnits = kPart / kOfWave, kUnitFragments = kOfWave / 16;
  int rows[kWaveUnits], first[kWaveUnits];  // of each: rows that exist, and the first one's number in the whole vocabulary
  bool all = true;
#pragma unroll
  for (int j = 0; j < kWaveUnits; ++j) {
    const int from = __builtin_amdgcn_readfirstlane(at * TL + part * kPart + j * kOfWave);
    const Unit u(pieces, ends, from / kUnitRows);
    rows[j] = u.rows - from % kUnitRows;
    first[j] = pieces.first[u.rank] + u.row + from % kUnitRows;
    all &= rows[j] >= kOfWave;
  }
  auto finish = [&](auto whole) {  // whole: none of the wave's rows is padding
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
    for (int r = 0; r < Product::FR; ++r) {
      const int n = Product::r_of(threadIdx.x, r);
      const bool live = n < tokens;
      const int label = live ? a.labels.get(a.token0 + n0 + n) : -1;
      bool here = false;
#pragma unroll
      for (int j = 0; j < kWaveUnits; ++j) here |= label >= first[j] && label < first[j] + min(rows[j], kOfWave);
      const bool any = __any(here);  // one wave in hundreds holds a label of its tokens
      const int kept = (MODE == kKeep || MODE == kGradient) && live ? a.pos ? a.pos[a.token0 + n0 + n] : n0 + n : -1;
      T* out = (T*)a.e + kept * ld + (int64_t)at * TL;
      // the wave's logits of the token, in fours: f(row in the unit, the unit's rows, the label's row in it, logits)
      auto each = [&](auto f) {
#pragma unroll
        for (int l = 0; l < Product::FL; ++l) {
          const int j = l / kUnitFragments;
          f(Product::l_of(threadIdx.x, l) - part * kPart - j * kOfWave, rows[j], label - first[j], acc[l][r]);
        }
      };
      // the same, and what f makes of them to G's row
      auto each_stored = [&](auto f) {
#pragma unroll
        for (int l = 0; l < Product::FL; l += 2) {
          typename Half<T>::x4 o[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int v = Product::l_of(threadIdx.x, l + k), j = (l + k) / kUnitFragments;
            o[k] = f(v - part * kPart - j * kOfWave, rows[j], label - first[j], acc[l + k][r]);
          }
          if (MODE == kKeep || MODE == kGradient) {
            const u32x4 row = Product::pair_up(o[0], o[1]);
            if (kept >= 0) *(u32x4*)(out + Product::l_of_pair(threadIdx.x, l)) = row;
          }
        }
      };
      if constexpr (MODE == kGradient) {
        const float lse = live ? a.lse[a.token0 + n0 + n] * kLog2e : 0.f, g = live ? a.upstream.get(a.token0 + n0 + n, label) * kUnit<T> : 0.f;
        each_stored([&](int row, int rows, int want, f32x4 z) {
          typename Half<T>::x4 o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p = exp2_of(__builtin_fmaf(z[i], kLog2e, -lse));
            if (any) p -= here && row + i == want ? 1.f : 0.f;
            o[i] = (T)((WHOLE || row + i < rows) && g != 0.f ? p * g : 0.f);
          }
          return o;
        });
      } else {
        float m = -INFINITY;
        each([&](int row, int rows, int, f32x4 z) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (WHOLE || row + i < rows) m = fmaxf(m, z[i]);
        });
        if (any) {
          float z_label = 0.f;
          bool found = false;
          each([&](int row, int rows, int want, f32x4 z) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (here && row + i == want && row + i < rows) z_label = z[i], found = true;
          });
          if (found) a.z_label[a.token0 + n0 + n] = z_label;
        }
        if constexpr (MODE == kLogits) {
#pragma unroll
          for (int l = 0; l < Product::FL; ++l) {
            const int v = Product::l_of(threadIdx.x, l), j = l / kUnitFragments, row = v - part * kPart - j * kOfWave;
            f32x4 z;
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = WHOLE || row + i < rows[j] ? acc[l][r][i] : -INFINITY;  // padding: probability 0
            if (live) *(f32x4*)((float*)a.e + (n0 + n) * ld + (int64_t)at * TL + v) = z;
          }
        }
#pragma unroll
        for (int d = 16; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
        m *= kLog2e;
        const float base = m == -INFINITY ? 0.f : m;  // a part of nothing but -inf has sum 0
        float sum = 0.f;
        each_stored([&](int row, int rows, int, f32x4 z) {
          typename Half<T>::x4 o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = WHOLE || row + i < rows ? exp2_of(__builtin_fmaf(z[i], kLog2e, -base)) : 0.f;
            sum += e;
            o[i] = (T)(e * kUnit<T>);
          }
          return o;
        });
        // inf - inf: a part with a logit of +inf has sum 1 at this maximum, and its other logits' E are 0, unless one is NaN
        if (__any(m == INFINITY)) {
          bool nan = false;
          each([&](int row, int rows, int, f32x4 z) {
#pragma unroll
            for (int i = 0; i < 4; ++i) nan |= (WHOLE || row + i < rows) && z[i] != z[i];
          });
          if (m == INFINITY) sum = nan ? NAN : 0.25f;
        }
#pragma unroll
        for (int d = 16; d < 64; d *= 2) sum += __shfl_xor(sum, d);
        if (live && lane < 16) a.stats[(n0 + n) * (pieces.columns() / kPart) + at * TL / kPart + part] = make_float2(m, sum);
      }
    }
  };
  if (all) finish(std::true_type());
  else finish(std::false_type());
}

template <class V, class F> __device__ __forceinline__ V block_reduce(V v, F f, V* shared) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = f(v, __shfl_xor(v, d));
  if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < (int)blockDim.x / 64; ++w) v = f(v, shared[w]);
  __syncthreads();
  return v;
}

// x with its rows on cache lines, a workgroup per row.
__global__ void __launch_bounds__(256) align_kernel(const char* x, int64_t x_stride, char* out, int64_t out_stride, int bytes) {
  for (int at = threadIdx.x * 16; at < bytes; at += 256 * 16) *(u32x4*)(out + blockIdx.x * out_stride + at) = *(const u32x4*)(x + blockIdx.x * x_stride + at);
}

struct TokenArgs {
  const float2* stats;
  int part;          // vocabulary of one entry
  int64_t token0;
  Labels labels;
  Upstream upstream;
  const float* z_label;
  float *lse, *loss;
  void* e;
  const float* logits;
  const int* pos;
  const char* x;
  int64_t x_stride, kept_stride, dx_stride;
  char *kept_x, *dx;   // [rows][hidden] for dw; and dx, where a token without a row has zeros
  int hidden;
  int tokens, second;  // kLogits: G's second rows begin at row `second`; rows between are zeros
  int given;           // kLogits: the lse is an input
};

// A workgroup per token: its parts' (m, sum) -> lse and loss, and with gradients its row of x, and of G: kKeep from E,
// in place; kLogits from the logits; kGradient: G is there and so is the lse.  Where tokens are few, several workgroups
// share one: each works out the lse for itself and takes gridDim.y'ths of the row, 4096 columns.  The token's statistics,
// 8 bytes for `part` rows, are then read twice by each of them, from cache: with 32 workgroups twice what they move.  With
// half and a quarter as many the kernel is longer all the same (1 token x 131072: 12.7 us, 13.5 and 15.7; 100 tokens 16.4,
// 16.5 and 17.2; 1 x 32768 7.0, 8.1 and 10.2).
// The label's own G = (p - 1) g comes from its logit in 32 bits: from a rounded p close to 1 next to nothing would be
// left of it.
template <class T, int MODE>
__global__ void __launch_bounds__(256) token_kernel(const Pieces pieces, const TokenArgs a) {
  __shared__ float shared[4];
  const int64_t ld = pieces.stride(), columns = pieces.columns(), at = a.token0 + blockIdx.x;
  const int parts = (int)(columns / a.part);
  const float2* stats = a.stats + (int64_t)blockIdx.x * parts;
  typedef typename Half<T>::x8 x8;
  if (MODE == kLogits && (int)blockIdx.x >= a.tokens) {
    for (int64_t v = (blockIdx.y * 256 + threadIdx.x) * 8; v < columns; v += gridDim.y * 256 * 8) *(x8*)((T*)a.e + blockIdx.x * ld + v) = x8{};
    return;
  }
  const int label = a.labels.get(at);
  const float z_label = label >= 0 ? a.z_label[at] : 0.f;
  float base, log_sum = 0.f, m = -INFINITY;  // lse is their sum, in units of log 2
  if (MODE == kGradient || (MODE == kLogits && a.given)) {
    base = a.lse[at] * kLog2e;
  } else {
    float sum = 0.f;
    for (int h = threadIdx.x; h < parts; h += 256) m = fmaxf(m, stats[h].x);
    m = block_reduce(m, [](float a, float b) { return fmaxf(a, b); }, shared);
    base = m == -INFINITY ? 0.f : m;
    for (int h = threadIdx.x; h < parts; h += 256) {
      const float2 s = stats[h];
      sum += s.y * exp2_of(s.x == base ? 0.f : s.x - base);  // (also where both are +inf)
    }
    sum = block_reduce(sum, [](float a, float b) { return a + b; }, shared);
    log_sum = log2f(sum);
    if (threadIdx.x == 0 && blockIdx.y == 0) {
      // in 64 bits, each rounded once; the loss not from the rounded lse, whose error may be larger than a small loss
      a.lse[at] = (float)(((double)base + log_sum) * kLn2);
      a.loss[at] = label == -1 ? 0.f : label < 0 ? NAN : (float)(((double)base - (double)z_label * kLog2e + log_sum) * kLn2);
    }
  }
  if constexpr (MODE != kStats) {
    const int row = a.pos ? a.pos[at] : (int)blockIdx.x;
    for (int d = (blockIdx.y * 256 + threadIdx.x) * 8; d < a.hidden; d += gridDim.y * 256 * 8) {
      if (row >= 0) *(x8*)(a.kept_x + row * a.kept_stride + d * 2) = label == -1 ? x8{} : *(const x8*)(a.x + blockIdx.x * a.x_stride + d * 2);
      else *(x8*)(a.dx + blockIdx.x * a.dx_stride + d * 2) = x8{};
    }
    if (MODE == kGradient || row < 0) return;
    const float g = a.upstream.get(at, label), lse2 = base + log_sum;
    int64_t want = -1;
    float of_label = 0.f;
    if (label >= 0) {
      const int r = Ends(pieces.first + 1, pieces.ranks).rank_of(label);
      want = (int64_t)pieces.unit0[r] * kUnitRows + label - pieces.first[r];
      of_label = expm1f((__builtin_fmaf(z_label, kLog2e, -base) - log_sum) * (float)kLn2) * g * kUnit<T>;
    }
    T* e = (T*)a.e + row * ld;
    for (int64_t v = (blockIdx.y * 256 + threadIdx.x) * 8; v < columns; v += gridDim.y * 256 * 8) {
      float p[8];
      if constexpr (MODE != kLogits) {
        const float top = stats[v / a.part].x;
        const float f = top == -INFINITY ? 0.f : exp2_of(top == lse2 ? 0.f : top - lse2) * g;  // (both may be +inf)
        const x8 kept = *(const x8*)(e + v);
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (float)kept[i] * f;
      } else {
        const float* z = a.logits + blockIdx.x * ld + v;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = exp2_of(__builtin_fmaf(z[i], kLog2e, -base) - log_sum) * (g * kUnit<T>);
      }
      x8 o, rest;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float whole = g == 0.f ? 0.f : v + i == want ? of_label : p[i];
        o[i] = (T)whole;
        rest[i] = (T)(whole - (float)o[i]);
      }
      *(x8*)(e + v) = o;
      if (MODE == kLogits) *(x8*)(e + a.second * ld + v) = rest;
    }
  }
}

struct SumsArgs {
  int64_t tokens;
  Labels labels;
  int mean;
  const float* rows;      // null: no loss
  float* loss;
  int gradients;          // what they are multiplied by is wanted
  const float* upstream;  // may be null where there is one for each of no tokens
  float* factor;          // null: one number for all tokens
  float unit;
  float* back;
};

struct OrderArgs {
  int64_t piece;  // tokens of a piece
  int *pos, *idx;  // a token's row among its piece's, -1: ignored; and the token (in the piece) of a row
  int* live;      // per piece: rows
};

// One workgroup over all tokens: the loss as one number, in 64 bits and in one order; with gradients what the products
// are multiplied by, max |g| (over the mean's count) over the unit, and with a number per token factor[n] = g[n] / max
// |g|.
__device__ __forceinline__ void sums_over_tokens(const SumsArgs& a, double* shared, int64_t kept = -1) {
  double sum = 0, count = 0;
  float top = 0.f;
  for (int64_t n = threadIdx.x; n < a.tokens; n += blockDim.x) {
    const int label = kept < 0 || a.factor ? a.labels.get(n) : 0;
    count += label != -1;
    if (a.rows) sum += a.rows[n];
    if (a.factor && label >= 0) {  // an infinite one is its token's own affair
      const float g = fabsf(a.upstream[n]);
      if (g < INFINITY) top = fmaxf(top, g);
    }
  }
  auto add = [](double a, double b) { return a + b; };
  auto counted = [&] { return kept >= 0 ? (double)kept : block_reduce(count, add, shared); };
  const double divisor = a.mean ? fmax(counted(), 1.0) : 1.0;
  if (a.rows) {
    sum = block_reduce(sum, add, shared);
    if (threadIdx.x == 0) *a.loss = (float)(sum / divisor);
  }
  if (!a.gradients) return;
  if (a.factor) {
    top = block_reduce(top, [](float a, float b) { return fmaxf(a, b); }, (float*)shared);
    for (int64_t n = threadIdx.x; n < a.tokens; n += blockDim.x) {
      const int label = a.labels.get(n);
      const float g = a.upstream[n];
      a.factor[n] = label == -1 ? 0.f : label < 0 ? NAN : g == 0.f ? 0.f : g / top;
    }
  } else {
    top = fabsf(*a.upstream);
    if (!(top < INFINITY) && counted() == 0.0) top = 0.f;  // zeros stay zeros
  }
  if (threadIdx.x == 0) *a.back = (float)((double)top / divisor / a.unit);
}

constexpr int kSumsThreads = 1024, kSumsWaves = kSumsThreads / 64;

// The rows of the tokens that are not ignored, in the tokens' order.  Each thread takes eight neighbours, so that a chunk
// of 8192 tokens waits for memory once.  -> how many there are
__device__ __forceinline__ int64_t order_tokens(const OrderArgs& o, int64_t tokens, const Labels& labels, int (*shared)[kSumsWaves]) {
  constexpr int kEach = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t kept = 0;
  int turn = 0;  // of the two halves of shared: whoever writes one again has met everyone at the other's barrier
  for (int64_t from = 0; from < tokens; from += o.piece) {
    const int64_t to = min(from + o.piece, tokens);
    int rows = 0;
    for (int64_t c = from; c < to; c += kSumsThreads * kEach, turn ^= 1) {
      const int64_t n = c + threadIdx.x * kEach;
      bool keep[kEach];
      int count = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) keep[j] = n + j < to && labels.get(n + j) != -1;
#pragma unroll
      for (int j = 0; j < kEach; ++j) count += keep[j];
      int upto = count;  // of the wave's threads up to this one, then of the waves
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
      }
      if (lane == 63) shared[turn][wave] = upto;
      __syncthreads();
      int waves = lane < kSumsWaves ? shared[turn][lane] : 0;
#pragma unroll
      for (int d = 1; d < kSumsWaves; d *= 2) {
        const int other = __shfl_up(waves, d);
        if (lane >= d) waves += other;
      }
      const int front = __shfl(waves, max(wave - 1, 0));
      int at = rows + (wave ? front : 0) + upto - count;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (n + j < to) o.pos[n + j] = keep[j] ? at : -1;
        if (keep[j]) o.idx[from + at++] = (int)(n + j - from);
      }
      rows += __shfl(waves, kSumsWaves - 1);
    }
    if (threadIdx.x == 0) o.live[from / o.piece] = rows;
    kept += rows;
  }
  return kept;
}

__global__ void __launch_bounds__(kSumsThreads) sums_kernel(const SumsArgs a, const OrderArgs o) {
  __shared__ double shared[kSumsWaves];
  __shared__ int counts[2][kSumsWaves];
  int64_t kept = -1;
  if (o.pos) kept = order_tokens(o, a.tokens, a.labels, counts);
  sums_over_tokens(a, shared, kept);
}

// The rows of all ranks' pieces as k of a product: a step is a unit.
struct PieceSource {
  static constexpr int further = 0;
  const Pieces* p;
  int64_t stride;
  int col_bytes, rank, units, left;  // units: of the rank, behind the step's
  const char* at;
  __device__ __forceinline__ PieceSource(const Pieces& pieces, int64_t stride, int col_bytes, int unit) : p(&pieces), stride(stride), col_bytes(col_bytes) {
    const Unit u(pieces, Ends(pieces.unit0 + 1, pieces.ranks), unit);
    rank = u.rank;
    units = pieces.unit0[rank + 1] - unit;
    at = pieces.w[rank] + (u.row - kUnitRows) * stride + col_bytes;
    left = u.rows + kUnitRows;
  }
  __device__ __forceinline__ void next() {
    if (units == 0) {
      while (rank + 1 < p->ranks && units == 0) {
        ++rank;
        units = p->unit0[rank + 1] - p->unit0[rank];
      }
      if (units) {
        at = p->w[rank] - kUnitRows * stride + col_bytes;
        left = p->rows[rank] + kUnitRows;
      }
    }
    --units;
    at += kUnitRows * stride;
    left -= kUnitRows;
  }
  __device__ __forceinline__ i32x4 base(int) const { return resource_at(at); }
};
static_assert(kUnitRows == kStepK, "a step of dx's product is a unit");

struct GradArgs {
  const void* g;     // [rows][stride]
  const char* x;     // the kept one
  const int *live, *idx;  // rows, and a row's token; null: all tokens, in order
  Labels labels;
  int64_t token0;
  int64_t x_stride, w_stride;
  int hidden, tokens, token_tiles, hidden_tiles;
  int second, rows;  // G's second rows begin at row `second` (0: there are none); rows of G in all
  int split_steps;   // dx: steps of kStepK for each part of the vocabulary
  float* parts;      // dx: [parts][rows][hidden]; null: dx itself is written
  int count;         // of parts
  int with_sums;     // dx: one workgroup more, for the sums over tokens
  int adders;        // dw: so many workgroups more, that add dx's parts
  int behind;        // they come last
  int share;         // lanes that share the parts of the same values
  char* dx;
  int64_t dx_stride, dw_stride;
  const float* back;
  float* sums;       // dw of the pieces so far, [tiles * kTile][hidden]; null: one piece
  int first, last;
};

template <class T> __device__ __forceinline__ typename Half<T>::x4 narrow(f32x4 v, float by) {
  typename Half<T>::x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)(v[i] * by);
  return o;
}

template <class T, class Shape>
__global__ void __launch_bounds__(Shape::kThreads, Shape::kWaves) dx_kernel(const Pieces pieces, const GradArgs a, const SumsArgs sums) {
  typedef typename Shape::template Product<T, true, false> Product;
  constexpr int TL = Shape::kL, TR = Shape::kR;
  __shared__ __attribute__((aligned(1024))) char smem[Product::kLdsBytes];
  if ((int)blockIdx.x == a.token_tiles * a.hidden_tiles * a.count) return sums_over_tokens(sums, (double*)smem);
  // All tiles of a part of the vocabulary follow each other in one XCD, which then reads the part of G and W once
  const int all = a.live ? *a.live : a.rows, token_tiles = (all + TR - 1) / TR, tiles = token_tiles * a.hidden_tiles;
  if ((int)blockIdx.x >= tiles * a.count) return;
  const int in_order = xcd_order(blockIdx.x, tiles * a.count), part = in_order / tiles;
  int tt, ht;
  tile_in_band(in_order % tiles, token_tiles, a.hidden_tiles, &tt, &ht);
  const int n0 = tt * TR, d0 = ht * TL, tokens = min(TR, all - n0), width = min(TL, a.hidden - d0);
  const int64_t ld = pieces.stride();
  const int step0 = part * a.split_steps, steps = min(a.split_steps, pieces.tiles * (kTile / kStepK) - step0);
  f32x4 acc[Product::FL][Product::FR] = {};
  {
    typename Product::LLanes ll;
    typename Product::RLanes rl;
    ll.place(threadIdx.x, a.w_stride, [&](int) { return width; });
    rl.place(threadIdx.x, ld * 2, [&](int i) { return tokens - i * kUnitRows; });
    Product::run(smem, steps, ll, PieceSource(pieces, a.w_stride, d0 * 2, step0), rl,
                 RowSource<TR>([&](int i) { return (const char*)a.g + ((n0 + i * kUnitRows) * ld + (int64_t)step0 * kStepK) * 2; }, steps * kStepK), acc);
  }
  const float back = a.parts ? 0.f : *a.back;  // (with parts the sums may still be under way)
#pragma unroll
  for (int r = 0; r < Product::FR; ++r) {
    const int n = Product::r_of(threadIdx.x, r);
    if (a.parts) {
#pragma unroll
      for (int l = 0; l < Product::FL; ++l) {
        const int d = Product::l_of(threadIdx.x, l);
        if (n < tokens && d < width) *(f32x4*)(a.parts + ((int64_t)part * a.rows + n0 + n) * a.hidden + d0 + d) = acc[l][r];
      }
    } else {
      const int64_t token = a.live && n < tokens ? a.idx[n0 + n] : n0 + n;
#pragma unroll
      for (int l = 0; l < Product::FL; l += 2) {
        const u32x4 row = Product::pair_up(narrow<T>(acc[l][r], back), narrow<T>(acc[l + 1][r], back));
        const int d = Product::l_of_pair(threadIdx.x, l);
        if (n < tokens && d < width) *(u32x4*)(a.dx + token * a.dx_stride + (d0 + d) * 2) = row;
      }
    }
  }
}

// dx from the parts of the vocabulary: four values at a time
template <class T> __device__ __forceinline__ void store_sum(const GradArgs& a, int64_t i, f32x4 sum, float back) {
  const int64_t row = i / a.hidden, token = a.live ? a.idx[row] : row;
  const bool ignored = !a.live && a.labels.get(a.token0 + token) == -1;  // (zero times what W holds, or times `back`, may be no zero)
  *(typename Half<T>::x4*)(a.dx + token * a.dx_stride + i % a.hidden * 2) = ignored ? typename Half<T>::x4{} : narrow<T>(sum, back);
}
template <class T> __device__ __forceinline__ void add_parts(const GradArgs& a, int adder) {
  const int64_t size = (int64_t)(a.live ? *a.live : a.tokens) * a.hidden, part = (int64_t)a.rows * a.hidden;
  const float back = *a.back;
  const int64_t thread = (int64_t)adder * blockDim.x + threadIdx.x, threads = (int64_t)a.adders * blockDim.x;
  if (a.share == 1) {
    for (int64_t i = thread * 4; i < size; i += threads * 4) {
      f32x4 sum = {}, rest = {};
      const float* from = a.parts + i;
#pragma unroll 8
      for (int p = 0; p < a.count; ++p, from += part) {
        sum += *(const f32x4*)from;
        if (a.second) rest += *(const f32x4*)(from + (int64_t)a.second * a.hidden);
      }
      store_sum<T>(a, i, sum + rest, back);
    }
    return;
  }
  // Where there are few values, lanes of a wave take turns at the parts of the same ones, so that none has many to wait
  // for (2 x 56079 x 576, 98 parts: dw 17.2 us, by one lane each 38.3).
  const int each = 64 / a.share, lane = threadIdx.x & 63;
  for (int64_t first = thread / 64 * each * 4; first < size; first += threads / 64 * each * 4) {
    const int64_t i = first + lane % each * 4;
    f32x4 sum = {}, rest = {};
    if (i < size) {
#pragma unroll 4
      for (int p = lane / each; p < a.count; p += a.share) {
        const float* from = a.parts + p * part + i;
        sum += *(const f32x4*)from;
        if (a.second) rest += *(const f32x4*)(from + (int64_t)a.second * a.hidden);
      }
    }
    sum += rest;
    for (int d = each; d < 64; d *= 2)
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += __shfl_xor(sum[k], d);
    if (i < size && lane < each) store_sum<T>(a, i, sum, back);
  }
}

template <class T, class Shape>
__global__ void __launch_bounds__(Shape::kThreads, Shape::kWaves) dw_kernel(const Pieces pieces, const Grads grads, const GradArgs a) {
  typedef typename Shape::template Product<T, true, true> Product;
  constexpr int TL = Shape::kL, TR = Shape::kR;
  __shared__ __attribute__((aligned(1024))) char smem[Product::kLdsBytes];
  const int adder = a.behind ? blockIdx.x - (gridDim.x - a.adders) : blockIdx.x, id = a.behind ? blockIdx.x : blockIdx.x - a.adders;
  if (adder >= 0 && adder < a.adders) return add_parts<T>(a, adder);
  int at, ht;
  tile_of(id, pieces.tiles * (kTile / TR), a.hidden_tiles, &at, &ht);
  const int d0 = ht * TL, width = min(TL, a.hidden - d0);
  const int64_t ld = pieces.stride();
  f32x4 acc[Product::FL][Product::FR] = {};
  {
    typename Product::LLanes ll;
    typename Product::RLanes rl;
    // x's rows once more for G's second rows: within a step, or behind the steps of the first
    ll.place(threadIdx.x, a.x_stride, [&](int) { return width; }, a.second && a.second < kStepK ? a.second : kStepK);
    rl.place(threadIdx.x, ld * 2, [&](int) { return TR; });
    const int all = a.live ? *a.live : a.rows;
    Product::run(smem, (all + kStepK - 1) / kStepK, ll, ColSource(a.x + d0 * 2, a.live ? all : a.tokens, a.x_stride, a.second >= kStepK), rl,
                 ColSource((const char*)a.g + (int64_t)at * TR * 2, all, ld * 2), acc);
  }
  static_assert(TR / Shape::kWavesR == kUnitRows, "a wave's rows are a unit");
  const int unit0 = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) / Shape::kWavesL);
  const Unit unit(pieces, Ends(pieces.unit0 + 1, pieces.ranks), at * (TR / kUnitRows) + unit0);
  const float back = *a.back;
#pragma unroll
  for (int r = 0; r < Product::FR; ++r) {
    const int at_tile = Product::r_of(threadIdx.x, r), v = at_tile - unit0 * kUnitRows;
    if (a.sums) {  // of the pieces of tokens so far
#pragma unroll
      for (int l = 0; l < Product::FL; ++l) {
        const int d = Product::l_of(threadIdx.x, l);
        f32x4* kept = (f32x4*)(a.sums + ((int64_t)at * TR + at_tile) * a.hidden + d0 + d);
        if (v >= unit.rows || d >= width) continue;
        if (!a.first) acc[l][r] += *kept;
        if (!a.last) *kept = acc[l][r];
      }
      if (!a.last) continue;
    }
#pragma unroll
    for (int l = 0; l < Product::FL; l += 2) {
      const u32x4 row = Product::pair_up(narrow<T>(acc[l][r], back), narrow<T>(acc[l + 1][r], back));
      const int d = Product::l_of_pair(threadIdx.x, l);
      if (v < unit.rows && d < width) *(u32x4*)(grads.dw[unit.rank] + (unit.row + v) * a.dw_stride + (d0 + d) * 2) = row;
    }
  }
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSCCLX_OK : fail(MSCCLX_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace
}  // namespace mscclx

using namespace mscclx;

struct mscclx_vocab_loss {
  mscclx_vocab_loss_desc desc;
  Pieces pieces;          // without pointers
  int64_t vocab = 0;
  int64_t piece = 0;      // tokens per piece
  uint64_t off_z = 0, off_loss = 0, off_factor = 0, off_back = 0, off_stats = 0, off_e = 0, off_sums = 0, off_parts = 0, off_logits = 0, off_x = 0, off_aligned = 0, off_pos = 0, off_idx = 0, off_live = 0, bytes = 0;
};

namespace {

// No C++ exception crosses the ABI.
template <class F> int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return MSCCLX_ERR_CAPACITY;
  } catch (...) {
    return MSCCLX_ERR_INVALID_ARG;
  }
}

int check_matrix(const char* what, const void* p, int64_t stride, int32_t hidden) {
  if (!p) return fail(MSCCLX_ERR_INVALID_ARG, std::string(what) + ": NULL");
  if ((uintptr_t)p % 16) return fail(MSCCLX_ERR_INVALID_ARG, std::string(what) + ": rows must start on 16-byte boundaries");
  if (stride < hidden || stride % 8 || stride > MSCCLX_VOCAB_LOSS_MAX_STRIDE)
    return fail(MSCCLX_ERR_INVALID_ARG, std::string(what) + ": the row stride must be a multiple of 8 elements, at least `hidden` and at most 2^22");
  return MSCCLX_OK;
}

// A matrix, or a vector as one row of it, that a call reads or writes.
struct Span {
  uintptr_t from;
  int64_t bytes, stride, rows;
  const char* what;
  int rank;
  bool written;
  uintptr_t to() const { return from + (rows - 1) * stride + bytes; }
};

// Two spans that share bytes, one of them written.  Matrices whose rows are equally far apart may lie side by
// side in one buffer.
bool collide(const Span& a, const Span& b) {
  if (!(a.written || b.written) || a.to() <= b.from || b.to() <= a.from) return false;
  if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) return true;
  if (a.rows <= 1 && b.rows <= 1) return true;
  const int64_t stride = a.rows > 1 ? a.stride : b.stride, off = (int64_t)((b.from - a.from) % stride + stride) % stride;
  return off < a.bytes || off + b.bytes > stride;
}

int check_spans(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  for (size_t i = 0; i < spans.size(); ++i)
    for (size_t j = i + 1; j < spans.size() && spans[j].from < spans[i].to(); ++j)
      if (collide(spans[i], spans[j])) {
        auto name = [](const Span& s) { return s.rank < 0 ? std::string(s.what) : std::string(s.what) + " of rank " + std::to_string(s.rank); };
        return fail(MSCCLX_ERR_ALIASED, name(spans[i]) + " and " + name(spans[j]) + " overlap, and one of them is written");
      }
  return MSCCLX_OK;
}

struct Call {
  Pieces pieces;
  Grads grads;
  Labels labels;
  float *z_label, *row_loss, *factor, *back, *sums, *parts, *logits;
  float2* stats;
  void* e;
  char *x, *aligned;
  OrderArgs order;
};

int check_call(const mscclx_vocab_loss* h, const mscclx_vocab_loss_io* io, bool forward, bool backward, Call* c) {
  if (!h || !io) return fail(MSCCLX_ERR_INVALID_ARG, "null argument");
  const mscclx_vocab_loss_desc& d = h->desc;
  if (backward && !d.gradients) return fail(MSCCLX_ERR_STATE, "the operator was created without gradients");
  if (io->tokens < 0 || io->tokens > d.max_tokens)
    return fail(MSCCLX_ERR_CAPACITY, std::to_string(io->tokens) + " tokens given, the operator was created for at most " + std::to_string(d.max_tokens));
  if (io->workspace_bytes < h->bytes)
    return fail(MSCCLX_ERR_CAPACITY, "workspace of " + std::to_string(io->workspace_bytes) + " bytes given, " + std::to_string(h->bytes) + " needed");
  if (!io->workspace || (uintptr_t)io->workspace % 256) return fail(MSCCLX_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
  c->pieces = h->pieces;
  const bool some = io->tokens > 0;
  int rc;
  if (some && (rc = check_matrix("x", io->x, io->x_stride, d.hidden))) return rc;
  if (!io->weights) return fail(MSCCLX_ERR_INVALID_ARG, "weights: NULL");
  for (int r = 0; r < d.ranks; ++r) {
    if (h->pieces.rows[r] && (rc = check_matrix(("weights of rank " + std::to_string(r)).c_str(), io->weights[r], io->weight_stride, d.hidden))) return rc;
    c->pieces.w[r] = (const char*)io->weights[r];
  }
  if (io->label_bytes != 4 && io->label_bytes != 8) return fail(MSCCLX_ERR_INVALID_ARG, "labels must be 32 or 64 bits wide");
  if (some && (!io->labels || (uintptr_t)io->labels % io->label_bytes)) return fail(MSCCLX_ERR_INVALID_ARG, "labels: NULL or not aligned to their type");
  if (some && (!io->lse || (uintptr_t)io->lse % 4)) return fail(MSCCLX_ERR_INVALID_ARG, "lse: NULL or not aligned to its type");
  if (forward && (some || d.reduction != MSCCLX_LOSS_NONE) && (!io->loss || (uintptr_t)io->loss % 4)) return fail(MSCCLX_ERR_INVALID_ARG, "loss: NULL or not aligned to its type");
  if (backward) {
    if ((some || d.reduction != MSCCLX_LOSS_NONE) && (!io->grad_loss || (uintptr_t)io->grad_loss % 4)) return fail(MSCCLX_ERR_INVALID_ARG, "grad_loss: NULL or not aligned to its type");
    if (some && (rc = check_matrix("dx", io->dx, io->dx_stride, d.hidden))) return rc;
    if (!io->dweights) return fail(MSCCLX_ERR_INVALID_ARG, "dweights: NULL");
    for (int r = 0; r < d.ranks; ++r) {
      if (h->pieces.rows[r] && (rc = check_matrix(("dweights of rank " + std::to_string(r)).c_str(), io->dweights[r], io->dweight_stride, d.hidden))) return rc;
      c->grads.dw[r] = (char*)io->dweights[r];
    }
  }
  std::vector<Span> spans;
  spans.reserve(2 * kMaxRanks + 8);
  auto use = [&](const char* what, const void* p, int64_t rows, int64_t columns, int64_t stride, int size, bool written, int rank = -1) {
    if (rows > 0 && columns > 0) spans.push_back({(uintptr_t)p, columns * size, stride * size, rows, what, rank, written});
  };
  const int64_t losses = d.reduction == MSCCLX_LOSS_NONE ? io->tokens : 1;
  use("the workspace", io->workspace, 1, (int64_t)h->bytes, 0, 1, true);
  use("x", io->x, io->tokens, d.hidden, io->x_stride, 2, false);
  use("labels", io->labels, 1, io->tokens, 0, io->label_bytes, false);
  use("lse", io->lse, 1, io->tokens, 0, 4, forward);
  if (forward) use("loss", io->loss, 1, losses, 0, 4, true);
  if (backward) use("grad_loss", io->grad_loss, 1, losses, 0, 4, false);
  if (backward) use("dx", io->dx, io->tokens, d.hidden, io->dx_stride, 2, true);
  for (int r = 0; r < d.ranks; ++r) {
    use("weights", io->weights[r], h->pieces.rows[r], d.hidden, io->weight_stride, 2, false, r);
    if (backward) use("dweights", io->dweights[r], h->pieces.rows[r], d.hidden, io->dweight_stride, 2, true, r);
  }
  if ((rc = check_spans(spans))) return rc;
  c->labels = Labels{io->labels, io->label_bytes == 8, d.ignore_index, h->vocab};
  char* ws = (char*)io->workspace;
  c->z_label = (float*)(ws + h->off_z);
  c->row_loss = d.reduction == MSCCLX_LOSS_NONE ? io->loss : (float*)(ws + h->off_loss);
  c->factor = (float*)(ws + h->off_factor);
  c->back = (float*)(ws + h->off_back);
  c->stats = (float2*)(ws + h->off_stats);
  c->e = ws + h->off_e;
  c->parts = (float*)(ws + h->off_parts);
  c->logits = (float*)(ws + h->off_logits);
  c->x = ws + h->off_x;
  c->aligned = ws + h->off_aligned;
  c->order = OrderArgs{h->piece, (int*)(ws + h->off_pos), (int*)(ws + h->off_idx), (int*)(ws + h->off_live)};
  c->sums = h->off_sums ? (float*)(ws + h->off_sums) : nullptr;
  return MSCCLX_OK;
}

constexpr int kLine = 128;
// Rows of the kept and of the aligned x begin on cache lines.
int64_t kept_stride(int hidden) { return ((int64_t)hidden * 2 + kLine - 1) / kLine * kLine; }

int tiles(int64_t n, int of = kTile) { return (int)((n + of - 1) / of); }

enum { kLarge, kMiddle, kSmall, kThin, kFew };
// Which shape a product takes.  Figures: us of the kernel with the shape / with the next best, by tokens x vocabulary x
// hidden in bf16, W from memory, all tiles in step.  Logits: Few in one round of its workgroups (128 x 8192 x 1024:
// 10.4 / 13.8 Small, 300 x 3000 x 4096 22 / 39, 512 x 4096 x 2048 21.5 / 23.6; 192 x 12000 x 1000, with 564, 25 / 18),
// two where W is read no more than twice (1 x 32768 x 4096: 80 / 101 Middle, 40 x 65536 x 4096 168 / 182; 128 x 65536 x
// 4096 245 / 187); Small while there are no more middle tiles than compute units (1113 x 2880 x 896: 15.7 / 18.2
// Middle, 600 x 3000 x 1000 17.2 / 20.6, 192 x 12000 x 1000 18.3 / 20.4; 353 x 18813 x 592, with 441, 26 / 21); Middle
// for as long as its tiles are one round (256 x 32768 x 2048: 60 / 73 Large, 300 x 20000 x 1024 23 / 31), Large from
// there on (171 x 34664 x 1640: 67 / 80 Middle, 1200 x 12000 x 4000 129 / 158, 500 x 32768 x 2048 74 / 97).
int64_t most_of_few(const Pieces& p) {
  const int columns = p.tiles * (kTile / Few::kL);
  return Few::kR * std::max(2 * kComputeUnits / columns, std::min(2, 4 * kComputeUnits / columns));
}
int logits_shape(const Pieces& p, int64_t tokens) {
  if (tokens <= most_of_few(p)) return kFew;
  const int64_t middle = (int64_t)tiles(tokens, Middle::kR) * p.tiles * (kTile / Middle::kL);
  return middle <= kComputeUnits ? kSmall : tokens <= 128 || middle <= 2 * kComputeUnits ? kMiddle : kLarge;
}
// A row of x that begins within a cache line has each step's 128 bytes in two; x is copied first where that is short
// against the product (forward and run in us, with the copy / without: 4096 x 32768 x 4104 908 / 982 and 3110 / 3210, 1500 x
// 40000 x 2008 249 / 263 and 762 / 779; near the border 1021 x 32003 x 1288 101 / 102 and 322 / 326, 1021 x 24000 x 1800 114 /
// 115 and 339 / 349, 1300 x 20000 x 2008 121 / 120 and 387 / 387, 1400 x 17000 x 2600 154 / 153 and 459 / 462; but 8192 x 8000
// x 904 148 / 145, 1200 x 12000 x 4000 105 / 102).  W's rows, which the same holds for, are read once: a copy of them would cost more.
bool align_pays(const Pieces& p, int64_t tokens, int hidden) {
  return p.tiles >= 64 && (int64_t)tiles(tokens) * p.tiles * tiles(hidden, kStepK) >= 40 * kComputeUnits;
}
// dw writes more than it reads where tokens are few; workgroups then hide each other's loads and stores (16 x 131072 x
// 4096: 222 Thin / 285 Large, 200 x 20000 x 3000 47 / 55, 300 x 20000 x 1024 25 / 28 Middle; 500 x 32768 x 2048 80 / 82
// Large, 1021 x 32003 x 1288 100 / 93).  More tokens: Large once its tiles fill the chip (1021 x 32003 x 1288: 93 / 110
// Middle; 1024 x 4096 x 512: 29 / 20 Middle).  How many of the tokens are ignored is known on the device only.
int dw_shape(const Pieces& p, int64_t tokens, int hidden) { return tokens <= 384 ? kThin : (int64_t)p.tiles * tiles(hidden) < kComputeUnits ? kMiddle : kLarge; }

// Logits in 32 bits and G twice where that decides about a rank's dw: with few tokens, or few for each rank.
bool is_wide(int64_t tokens, int ranks) { return tokens <= 32 || (tokens <= kWideTokens && tokens < 16 * ranks); }
int64_t most_wide(int64_t tokens, int ranks) { return std::min<int64_t>(tokens, std::max(32, std::min(kWideTokens, 16 * ranks - 1))); }
// Where G's second rows begin, so that no step of dw's product and no tile of dx's has more of them than need be; rows
// behind the first ones are zeros.
int second_row(int64_t tokens) { return tokens <= 16 ? 16 : tokens <= 32 ? 32 : (int)((tokens + kStepK - 1) / kStepK * kStepK); }

// dx: the shape, and into how many parts the vocabulary is cut so that the last round of tiles fills the chip, by what
// each would take: rounds of the slots, each of split_steps steps and 6 us around them, and the parts written and added.
// A step takes 1.25 us in Large, 0.9 in Middle with two workgroups on a unit (1.5 in a long product, which slows the clock,
// but then for both).  By tokens x vocabulary x hidden: 4096 x 32768 x 4104, 272 large tiles, 1100 us and 70 to add in four
// parts, 1625 in one; 6000 x 8000 x 3504, 336 large tiles, 340 in one part, 306 and 84 to add in two.  412 x 21975 x 2512:
// Large 54 us / Middle 60, 1021 x 32003 x 1288 79 / 98, 353 x 18813 x 592 24 / 18, 8192 x 2048 x 1024 45 / 37.  No part has
// less than eight steps (the adding is dw's: with four, 1024 x 4096 x 512 takes 3 us longer there).  Large not where most
// of its tile would be empty (64 x 131072 x 4096: 209 / 203 Middle).  Few where all is a few microseconds, as long as W,
// which it reads again for every 32 tokens, is small (1 x 8192 x 1024: 7.4 us / 10.5 Middle, 128 x 8192 x 1024 12.2 / 13.9;
// 1 x 32768 x 2048 26.6 / 24.8, 40 x 65536 x 4096 139 / 105).
struct DxPlan {
  int shape, token_tiles, hidden_tiles, parts, split_steps;
  bool separate;  // the parts are kept and added
};
DxPlan dx_plan(const Pieces& p, int64_t tokens, int hidden, bool separate) {
  const int steps = p.tiles * (kTile / kStepK);
  const int64_t w_reads = (int64_t)tiles(tokens, Few::kR) * p.tiles * kTile * hidden * 2;
  // one part in 32 bits, written and read; the same for 32 counts of tokens, as all of a plan is
  const double part_us = (double)tiles(tokens, 32) * 32 * hidden * 8 / 3.5e6;
  DxPlan best;
  double best_us = INFINITY;
  auto consider = [&](int shape, int l, int r, int slots, double step_us, bool fill_once) {
    const int64_t token_tiles = tiles(tokens, r), hidden_tiles = tiles(hidden, l), all = token_tiles * hidden_tiles;
    for (int64_t parts = 1; parts == 1 || (parts <= steps / 8 && all * parts <= (fill_once ? 1 : 16) * slots); ++parts) {
      const int split_steps = (int)((steps + parts - 1) / parts);
      if ((steps + split_steps - 1) / split_steps != parts) continue;
      const bool kept = separate || parts > 1;
      const double us = (double)((all * parts + slots - 1) / slots) * (split_steps * step_us + 6) + (kept ? parts * part_us : 0);
      if (us < best_us) best_us = us, best = DxPlan{shape, (int)token_tiles, (int)hidden_tiles, (int)parts, split_steps, kept};
    }
  };
  if (tokens <= 256 && w_reads <= 96 << 20) {
    consider(kFew, Few::kL, Few::kR, 2 * kComputeUnits, 0.5, true);
  } else {
    consider(kMiddle, Middle::kL, Middle::kR, 2 * kComputeUnits, 0.9, false);
    if (tokens > 96) consider(kLarge, Large::kL, Large::kR, kComputeUnits, 1.25, false);
  }
  return best;
}

template <class T, int MODE>
int launch_logits(int shape, const Pieces& p, LogitsArgs& a, hipStream_t stream) {
  auto go = [&](auto s) {
    typedef decltype(s) S;
    a.token_tiles = tiles(a.tokens, S::kR);
    const int grid = a.token_tiles * p.tiles * (kTile / S::kL);
    // In step, all workgroups ask for the same 128 bytes of each row of W at a time.  Where rows lie a multiple of 4 KiB
    // apart those are in few of memory's channels, so every eight tiles begin at another k (128 x 65536 x 4096: 146 us, in
    // step 175; 256 x 32768 x 2048 51 / 59, 500 x 32768 x 2048 68 / 79; not with so many tokens that W's reads hide, 4096 x
    // 32768 x 4096 850 / 841, nor with one tile of a few, 16 x 131072 x 4096 264 / 256).  With one workgroup of Few per
    // compute unit each begins at its own (the loss of 1 token x 32768 x 2048: 32.2 us, in step 36.2).
    a.apart = S::kR == Few::kR && grid <= kComputeUnits ? 1 : a.tokens > Few::kR && a.tokens <= 2048 && a.w_stride % 4096 == 0 ? 8 : 0;
    hipLaunchKernelGGL((logits_kernel<T, MODE, S>), dim3((unsigned)grid), dim3(S::kThreads), 0, stream, p, a);
    return launched("logits_kernel");
  };
  if constexpr (MODE != kLogits)  // (up to kWideTokens tokens)
    if (shape == kLarge) return go(Large());
  return shape == kMiddle ? go(Middle()) : shape == kSmall ? go(Small()) : go(Few());
}

template <class T>
int enqueue(const mscclx_vocab_loss* h, const mscclx_vocab_loss_io* io, bool forward, bool backward, const Call& c, hipStream_t stream) {
  const mscclx_vocab_loss_desc& d = h->desc;
  const Pieces& p = c.pieces;
  const int64_t n = io->tokens;
  const int mean = d.reduction == MSCCLX_LOSS_MEAN, per_token = d.reduction == MSCCLX_LOSS_NONE;
  const Upstream upstream = {io->grad_loss, per_token ? c.factor : nullptr};
  int rc;
  const bool wide = backward && is_wide(n, d.ranks);
  // The sums over tokens: for the gradients in front of everything, unless that is one number and nothing in front of
  // the products asks for it; for the loss as one number behind the last piece's tokens (beside its gradients, where dx
  // has parts). Up to kWideTokens tokens, rows of zeros cost less than the launch that finds out which they are
  const bool ordered = backward && n > kWideTokens;
  const bool early = backward && (per_token || !forward || ordered);
  SumsArgs first = {n, c.labels, mean, nullptr, nullptr, 1, io->grad_loss, per_token ? c.factor : nullptr, kUnit<T>, c.back};
  SumsArgs totals = {n, c.labels, mean, forward && !per_token ? c.row_loss : nullptr, io->loss, backward && !early, io->grad_loss, nullptr, kUnit<T>, c.back};
  auto sums = [&](const SumsArgs& what, const OrderArgs& order) {
    hipLaunchKernelGGL(sums_kernel, dim3(1), dim3(kSumsThreads), 0, stream, what, order);
    return launched("sums_kernel");
  };
  if (early && (rc = sums(first, ordered ? c.order : OrderArgs{}))) return rc;
  const int64_t all = std::max<int64_t>(n, backward ? 1 : 0);  // no tokens: dw is still written, with zeros
  for (int64_t at = 0; at < all; at += h->piece) {
    const int now = (int)std::min(h->piece, n - at);
    const bool last = at + now >= n;
    LogitsArgs a = {};
    a.x = (const char*)io->x + at * io->x_stride * 2;
    a.x_stride = io->x_stride * 2;
    a.w_stride = io->weight_stride * 2;
    a.hidden = d.hidden;
    a.tokens = now;
    a.token0 = at;
    a.labels = c.labels;
    a.upstream = upstream;
    a.pos = ordered ? c.order.pos : nullptr;
    a.stats = c.stats;
    a.z_label = c.z_label;
    a.e = c.e;
    a.lse = io->lse;
    if (now > 0) {
      const int shape = logits_shape(p, now);
      if (shape == kLarge && ((uintptr_t)a.x | a.x_stride) % kLine && align_pays(p, now, d.hidden)) {
        hipLaunchKernelGGL(align_kernel, dim3(now), dim3(256), 0, stream, a.x, a.x_stride, c.aligned, kept_stride(d.hidden), d.hidden * 2);
        if ((rc = launched("align_kernel"))) return rc;
        a.x = c.aligned;
        a.x_stride = kept_stride(d.hidden);
      }
      if (wide) a.e = c.logits;
      if ((rc = wide ? launch_logits<T, kLogits>(shape, p, a, stream) : !forward ? launch_logits<T, kGradient>(shape, p, a, stream) : backward ? launch_logits<T, kKeep>(shape, p, a, stream) : launch_logits<T, kStats>(shape, p, a, stream)))
        return rc;
      TokenArgs t = {};
      t.stats = c.stats;
      t.part = shape == kLarge ? Large::kL / Large::kWavesL : shape == kFew ? Few::kL / Few::kWavesL : Middle::kL / Middle::kWavesL;
      static_assert(Small::kL / Small::kWavesL == Middle::kL / Middle::kWavesL, "their entries are of as much vocabulary");
      t.token0 = at;
      t.labels = c.labels;
      t.upstream = upstream;
      t.z_label = c.z_label;
      t.lse = io->lse;
      t.loss = c.row_loss;
      t.e = c.e;
      t.logits = c.logits;
      t.pos = a.pos;
      t.x = (const char*)io->x + at * io->x_stride * 2;
      t.x_stride = io->x_stride * 2;
      t.kept_x = c.x;
      t.kept_stride = kept_stride(d.hidden);
      t.dx = (char*)io->dx + at * io->dx_stride * 2;
      t.dx_stride = io->dx_stride * 2;
      t.hidden = d.hidden;
      t.tokens = now;
      t.second = second_row(now);
      t.given = !forward;
      const unsigned slices = (unsigned)std::max(1, std::min(4 * kComputeUnits / now, p.tiles * kTile / 4096));
      if (wide) hipLaunchKernelGGL((token_kernel<T, kLogits>), dim3(t.second, slices), dim3(256), 0, stream, p, t);
      else if (!forward) hipLaunchKernelGGL((token_kernel<T, kGradient>), dim3(now), dim3(256), 0, stream, p, t);
      else if (backward) hipLaunchKernelGGL((token_kernel<T, kKeep>), dim3(now, slices), dim3(256), 0, stream, p, t);
      else hipLaunchKernelGGL((token_kernel<T, kStats>), dim3(now), dim3(256), 0, stream, p, t);
      if ((rc = launched("token_kernel"))) return rc;
    }
    const bool behind = last && forward && !per_token;  // the sums come now
    const int second = wide && now > 0 ? second_row(now) : 0, rows = second + now;
    const DxPlan plan = backward && now > 0 ? dx_plan(p, rows, d.hidden, !ordered) : DxPlan{};
    if (behind && !plan.separate && (rc = sums(totals, OrderArgs{}))) return rc;
    if (!backward) continue;
    GradArgs g = {};
    g.g = c.e;
    g.x = c.x;
    g.x_stride = kept_stride(d.hidden);
    if (ordered) g.live = c.order.live + at / h->piece, g.idx = c.order.idx + at;
    g.labels = c.labels;
    g.token0 = at;
    g.w_stride = a.w_stride;
    g.hidden = d.hidden;
    g.tokens = now;
    g.second = second;
    g.rows = rows;
    g.dx = (char*)io->dx + at * io->dx_stride * 2;
    g.dx_stride = io->dx_stride * 2;
    g.dw_stride = io->dweight_stride * 2;
    g.back = c.back;
    g.sums = n > h->piece ? c.sums : nullptr;
    g.first = at == 0;
    g.last = last;
    if (now > 0) {
      g.token_tiles = plan.token_tiles;
      g.hidden_tiles = plan.hidden_tiles;
      g.split_steps = plan.split_steps;
      g.parts = plan.separate ? c.parts : nullptr;
      g.count = plan.parts;
      g.with_sums = g.parts && behind;
      auto go = [&](auto s) {
        typedef decltype(s) S;
        hipLaunchKernelGGL((dx_kernel<T, S>), dim3((unsigned)(g.token_tiles * g.hidden_tiles * plan.parts + g.with_sums)), dim3(S::kThreads), 0, stream, p, g, totals);
        return launched("dx_kernel");
      };
      if ((rc = plan.shape == kLarge ? go(LargeDx()) : plan.shape == kMiddle ? go(Middle()) : go(Few()))) return rc;
    }
    auto go = [&](auto s) {
      typedef decltype(s) S;
      g.hidden_tiles = tiles(d.hidden, S::kL);
      g.share = 1;
      while (g.share < 16 && g.share < g.count && (int64_t)now * d.hidden / 4 * g.share < kComputeUnits * 128) g.share *= 2;
      g.adders = g.parts ? (int)std::min<int64_t>(2 * kComputeUnits, ((int64_t)now * d.hidden / 4 * g.share + S::kThreads - 1) / S::kThreads) : 0;
      const int all_tiles = p.tiles * (kTile / S::kR) * g.hidden_tiles, slots = kComputeUnits * 4 * S::kWaves / (S::kThreads / 64);
      // In front they have done when the last tiles take the chip for themselves (2048 x 32768 x 2048: dw 260 us, behind
      // 266; 64 x 20000 x 2048 21.5 / 23.4); but where all tiles have a place at once none waits for them (1113 x 2880 x
      // 896: 24.2 in front, 17.0 behind).
      g.behind = all_tiles <= slots;
      hipLaunchKernelGGL((dw_kernel<T, S>), dim3((unsigned)(g.adders + all_tiles)), dim3(S::kThreads), 0, stream, p, c.grads, g);
      return launched("dw_kernel");
    };
    const int shape = dw_shape(p, now, d.hidden);
    if ((rc = shape == kLarge ? go(Large()) : shape == kMiddle ? go(Middle()) : go(Thin()))) return rc;
  }
  if (n == 0 && forward && !per_token && !backward) return sums(totals, OrderArgs{});
  return MSCCLX_OK;
}

int call(const mscclx_vocab_loss* h, const mscclx_vocab_loss_io* io, bool forward, bool backward, void* stream) {
  return guarded([&] {
    Call c = {};
    if (int rc = check_call(h, io, forward, backward, &c)) return rc;
    return h->desc.dtype == MSCCLX_BF16 ? enqueue<__bf16>(h, io, forward, backward, c, (hipStream_t)stream)
                                        : enqueue<_Float16>(h, io, forward, backward, c, (hipStream_t)stream);
  });
}

}  // namespace

extern "C" {

int mscclx_vocab_loss_create(const mscclx_vocab_loss_desc* desc, mscclx_vocab_loss** out, uint64_t* workspace_bytes, int64_t* piece_tokens) {
  return guarded([&] {
    if (!desc || !out) return fail(MSCCLX_ERR_INVALID_ARG, "null argument");
    *out = nullptr;
    const mscclx_vocab_loss_desc& d = *desc;
    if (d.ranks < 1 || d.ranks > kMaxRanks) return fail(MSCCLX_ERR_INVALID_ARG, "between 1 and " + std::to_string(kMaxRanks) + " ranks");
    if (!d.rank_rows) return fail(MSCCLX_ERR_INVALID_ARG, "rank_rows: NULL");
    if (d.dtype != MSCCLX_BF16 && d.dtype != MSCCLX_F16) return fail(MSCCLX_ERR_UNSUPPORTED, "the vocabulary loss takes bfloat16 and float16");
    if (d.hidden < 8 || d.hidden % 8 || d.hidden > MSCCLX_VOCAB_LOSS_MAX_STRIDE) return fail(MSCCLX_ERR_INVALID_ARG, "hidden must be a positive multiple of 8, at most 2^22");
    if (d.reduction < MSCCLX_LOSS_NONE || d.reduction > MSCCLX_LOSS_MEAN) return fail(MSCCLX_ERR_INVALID_ARG, "unknown reduction");
    if (d.max_tokens < 0 || d.max_tokens > (1ll << 31) - 1) return fail(MSCCLX_ERR_INVALID_ARG, "max_tokens must be between 0 and 2^31 - 1");
    mscclx_vocab_loss* h = new mscclx_vocab_loss();
    h->desc = d;
    h->desc.rank_rows = nullptr;
    Pieces& p = h->pieces;
    p.ranks = d.ranks;
    int units = 0;
    for (int r = 0; r < d.ranks; ++r) {
      const int64_t rows = d.rank_rows[r];
      if (rows < 0 || rows > MSCCLX_VOCAB_LOSS_MAX_STRIDE || (int64_t)units * kUnitRows + rows > MSCCLX_VOCAB_LOSS_MAX_STRIDE - kTile) {  // (rows of G are addressed with 32-bit offsets, 64 at a time)
        delete h;
        return fail(MSCCLX_ERR_INVALID_ARG, "the ranks' rows must not be negative and, each rank's rounded up to 64, add up to less than 2^22");
      }
      p.rows[r] = (int)rows;
      p.first[r] = (int)h->vocab;
      p.unit0[r] = units;
      units += tiles(rows, kUnitRows);
      h->vocab += rows;
    }
    p.unit0[d.ranks] = units;
    p.first[d.ranks] = (int)h->vocab;
    p.tiles = tiles((int64_t)units * kUnitRows);
    if (h->vocab == 0) {
      delete h;
      return fail(MSCCLX_ERR_INVALID_ARG, "the vocabulary is empty");
    }
    const uint64_t row = (uint64_t)p.stride() * 2;  // bytes of E for a token
    const uint64_t budget = d.piece_bytes ? d.piece_bytes : MSCCLX_VOCAB_LOSS_PIECE_BYTES;
    const int64_t fit = (int64_t)(budget / ((uint64_t)p.columns() * 2) / kTile * kTile);
    h->piece = std::max<int64_t>(1, std::min<int64_t>(d.max_tokens, std::max<int64_t>(kTile, std::min<int64_t>(fit, 1 << 20))));
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
      const uint64_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    const uint64_t n = (uint64_t)d.max_tokens;
    h->off_back = take(4);
    h->off_z = take(n * 4);
    h->off_loss = take(n * 4);
    h->off_factor = take(n * 4);
    h->off_pos = take(n * 4);
    h->off_idx = take(n * 4);
    h->off_live = take((n / h->piece + 1) * 4);
    h->off_x = d.gradients ? take((uint64_t)h->piece * kept_stride(d.hidden)) : 0;
    h->off_aligned = align_pays(p, h->piece, d.hidden) ? take((uint64_t)h->piece * kept_stride(d.hidden)) : 0;
    const uint64_t wide = (uint64_t)p.tiles * kTile;
    h->off_stats = take(std::max(std::min<uint64_t>(h->piece, most_of_few(p)) * (wide / (Few::kL / Few::kWavesL)), (uint64_t)h->piece * (wide / (Middle::kL / Middle::kWavesL))) * sizeof(float2));
    const uint64_t wide_rows = most_wide(d.max_tokens, d.ranks);
    h->off_logits = d.gradients ? take(wide_rows * p.stride() * 4) : 0;
    h->off_e = d.gradients ? take(std::max<uint64_t>(h->piece, second_row(wide_rows) + wide_rows) * row) : 0;
    h->off_sums = d.gradients && d.max_tokens > h->piece ? take((uint64_t)p.tiles * kTile * d.hidden * 4) : 0;
    uint64_t parts = 0;  // dx's parts at the token count that needs most of them
    auto need = [&](int64_t rows, bool separate) {
      const DxPlan plan = dx_plan(p, rows, d.hidden, separate);
      if (plan.separate) parts = std::max(parts, (uint64_t)plan.parts * rows * d.hidden * 4);
    };
    for (int64_t t = 1; d.gradients && t <= std::min<int64_t>(h->piece, kWideTokens); ++t) need(is_wide(t, d.ranks) ? second_row(t) + t : t, true);
    for (int64_t t = 32; d.gradients && t - 31 <= h->piece; t += 32) need(std::min(t, h->piece), false);  // (the plan is the same from t - 31 on)
    h->off_parts = take(parts);
    h->bytes = at;
    if (workspace_bytes) *workspace_bytes = at;
    if (piece_tokens) *piece_tokens = h->piece;
    *out = h;
    return (int)MSCCLX_OK;
  });
}

int mscclx_vocab_loss_destroy(mscclx_vocab_loss* loss) {
  delete loss;
  return MSCCLX_OK;
}

int mscclx_vocab_loss_forward(const mscclx_vocab_loss* loss, const mscclx_vocab_loss_io* io, void* stream) { return call(loss, io, true, false, stream); }
int mscclx_vocab_loss_backward(const mscclx_vocab_loss* loss, const mscclx_vocab_loss_io* io, void* stream) { return call(loss, io, false, true, stream); }
int mscclx_vocab_loss_run(const mscclx_vocab_loss* loss, const mscclx_vocab_loss_io* io, void* stream) { return call(loss, io, true, true, stream); }

}  // extern "C"
