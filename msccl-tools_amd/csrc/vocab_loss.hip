// Softmax cross entropy over a vocabulary that is cut into the ranks' pieces, with its gradients, without keeping the logits.
//
//   z[n][v]  = sum over d of x[n][d] w[v][d]        w: the ranks' rows one under the other
//   lse[n]   = log sum over v of exp z[n][v],   loss[n] = lse[n] - z[n][label[n]]
//   G[n][v]  = g[n] (exp(z[n][v] - lse[n]) - [v = label[n]]),   dx = G w,   dw = transposed(G) x
//
// Tokens go through in pieces of at most `piece` rows; per piece, three products on the matrix cores (tile_product.h):
//   logits   z of a tile of vocabulary x tokens stays in registers; what leaves are, for each token and each half tile of the
//            vocabulary, the maximum m and the sum of exp(z - m), and with gradients E = exp(z - m) in 16 bits;
//   join     the pieces' (m, sum) become the token's lse;
//   scale    E becomes G in place: G = (E exp(m - lse) - [label]) g / max|g|;
//   dx, dw   the two products, on G.
// The 16-bit E and G are what the matrix cores take.  Both are rounded relative to their own size (bf16 2^-9 on average, as the outputs
// are), with 2^15 as unit in fp16, so that probabilities down to 2^-29 are normal numbers; |g| is divided by its largest value for
// the same reason and multiplied back in 32 bits behind the products.
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
constexpr int kTile = 256;              // vocabulary, tokens and hidden of a workgroup's tile
constexpr float kLog2e = 1.4426950408889634f;

// The ranks' pieces of the vocabulary, passed to the kernels by value.  Tiles of kTile rows; none spans two ranks.
struct Pieces {
  int ranks, tiles;
  int rows[kMaxRanks];
  int tile0[kMaxRanks + 1];  // the rank's first tile
  int first[kMaxRanks];      // the rank's first row in the whole vocabulary
  const char* w[kMaxRanks];
  __device__ __forceinline__ int rank_of(int tile) const {
    int r = 0;
    while (r + 1 < ranks && tile >= tile0[r + 1]) ++r;
    return r;
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

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
template <class T> constexpr float kUnit = std::is_same_v<T, _Float16> ? 32768.0f : 1.0f;

enum { kStats = 0, kKeep = 1, kGradient = 2 };

struct LogitsArgs {
  const char* x;
  int64_t x_stride;  // bytes
  int64_t w_stride;
  int hidden, tokens, token_tiles;
  int64_t token0;    // of the labels, lse and factor
  Labels labels;
  float2* stats;     // [2 * tiles][ld_stats]
  int64_t ld_stats;
  float* z_label;
  void* e;           // [tokens][tiles * kTile]
  const float* lse;
  const float* factor;
};

// Tiles in an order that keeps the workgroups of one XCD (every eighth of the grid) on neighbouring tiles: columns of
// up to eight row tiles share what they read.
__device__ __forceinline__ void tile_of(int id, int rows, int cols, int* row, int* col) {
  const int total = rows * cols, per = total / 8;
  if (id < per * 8) id = id % 8 * per + id / 8;
  const int band = 8 * cols, at = id / band * 8, high = min(8, rows - at), in = id % band;
  *row = at + in % high;
  *col = in / high;
}

template <class T, int MODE>
__global__ void __launch_bounds__(512, 2) logits_kernel(const Pieces pieces, const LogitsArgs a) {
  typedef TileProduct<T, kTile, kTile, 2, 4, false, false> Product;
  __shared__ __attribute__((aligned(1024))) char smem[Product::kLdsBytes];
  int tt, vt;
  tile_of(blockIdx.x, a.token_tiles, pieces.tiles, &tt, &vt);
  const int rank = pieces.rank_of(vt), row0 = (vt - pieces.tile0[rank]) * kTile, rows = min(kTile, pieces.rows[rank] - row0);
  const int n0 = tt * kTile, tokens = min(kTile, a.tokens - n0);
  f32x4 acc[Product::FL][Product::FR] = {};
  {
    typename Product::LLanes ll;
    typename Product::RLanes rl;
    ll.place(threadIdx.x, a.w_stride, rows);
    rl.place(threadIdx.x, a.x_stride, tokens);
    Product::run(smem, (a.hidden + kStepK - 1) / kStepK, ll, RowSource{pieces.w[rank] + row0 * a.w_stride, a.hidden}, rl,
                 RowSource{a.x + n0 * a.x_stride, a.hidden}, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l0 = wave % 2 * 128, r0 = wave / 2 * 64;
  const int64_t ld = (int64_t)pieces.tiles * kTile;
  const int v0 = l0 + (lane >> 4) * 4;  // + 16 * l + i
#pragma unroll
  for (int r = 0; r < Product::FR; ++r) {
    const int n = r0 + r * 16 + (lane & 15);
    const bool live = n < tokens;
    const int label = live ? a.labels.get(a.token0 + n0 + n) : -1;
    const int want = label >= 0 ? label - pieces.first[rank] - row0 : -1;
    typename Half<T>::x4* out = (typename Half<T>::x4*)((T*)a.e + (n0 + n) * ld + (int64_t)vt * kTile + v0);
    if constexpr (MODE == kGradient) {
      const float lse = live ? a.lse[a.token0 + n0 + n] : 0.f, g = live ? a.factor[a.token0 + n0 + n] * kUnit<T> : 0.f;
#pragma unroll
      for (int l = 0; l < Product::FL; ++l) {
        typename Half<T>::x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = v0 + l * 16 + i;
          const float p = exp_of(acc[l][r][i] - lse) - (v == want ? 1.f : 0.f);
          o[i] = (T)(v < rows && g != 0.f ? p * g : 0.f);
        }
        if (live) out[l * 4] = o;
      }
    } else {
      float m = -INFINITY, z_label = 0.f;
      bool found = false;
#pragma unroll
      for (int l = 0; l < Product::FL; ++l)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = v0 + l * 16 + i;
          if (v == want && v < rows) z_label = acc[l][r][i], found = true;
          if (v >= rows) acc[l][r][i] = -INFINITY;
          m = fmaxf(m, acc[l][r][i]);
        }
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const float base = m == -INFINITY ? 0.f : m;  // a half tile of nothing but -inf has sum 0
      float sum = 0.f;
#pragma unroll
      for (int l = 0; l < Product::FL; ++l) {
        typename Half<T>::x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = exp_of(acc[l][r][i] - base);
          sum += e;
          o[i] = (T)(e * kUnit<T>);
        }
        if (MODE == kKeep && live) out[l * 4] = o;
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (live) {
        if (lane < 16) a.stats[(int64_t)(2 * vt + wave % 2) * a.ld_stats + n0 + n] = make_float2(m, sum);
        if (found) a.z_label[a.token0 + n0 + n] = z_label;
      }
    }
  }
}

// (m, sum) of all half tiles -> lse and loss of 32 tokens; eight threads per token
__global__ void __launch_bounds__(256) join_kernel(const float2* stats, int64_t ld_stats, int halves, int tokens, int64_t token0, Labels labels,
                                                   const float* z_label, float* lse, float* loss) {
  __shared__ float2 part[8][32];
  const int n = blockIdx.x * 32 + threadIdx.x % 32, g = threadIdx.x / 32;
  float m = -INFINITY, sum = 0.f;
  if (n < tokens)
    for (int h = g; h < halves; h += 8) {
      const float2 s = stats[(int64_t)h * ld_stats + n];
      const float top = fmaxf(m, s.x);
      if (top == -INFINITY) sum += s.y;  // nothing yet: s.y is 0 or NaN
      else sum = sum * exp_of(m - top) + s.y * exp_of(s.x - top);
      m = top;
    }
  part[g][threadIdx.x % 32] = make_float2(m, sum);
  __syncthreads();
  if (g == 0 && n < tokens) {
    for (int i = 1; i < 8; ++i) {
      const float2 s = part[i][threadIdx.x];
      const float top = fmaxf(m, s.x);
      if (top == -INFINITY) sum += s.y;
      else sum = sum * exp_of(m - top) + s.y * exp_of(s.x - top);
      m = top;
    }
    const int64_t at = token0 + n;
    const float v = m + logf(sum);
    lse[at] = v;
    const int label = labels.get(at);
    loss[at] = label == -1 ? 0.f : label < 0 ? NAN : v - z_label[at];
  }
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

// the tokens' losses to one number, in 64 bits and in one order
__global__ void __launch_bounds__(1024) total_kernel(const float* rows, int64_t tokens, Labels labels, int mean, float* loss) {
  __shared__ double shared[16];
  double sum = 0, count = 0;
  for (int64_t n = threadIdx.x; n < tokens; n += 1024) {
    sum += rows[n];
    count += labels.get(n) != -1;
  }
  auto add = [](double a, double b) { return a + b; };
  sum = block_reduce(sum, add, shared);
  count = block_reduce(count, add, shared);
  if (threadIdx.x == 0) *loss = (float)(mean ? sum / fmax(count, 1.0) : sum);
}

// factor[n] = g[n] / max |g| and behind the factors, in back[0], what the products are multiplied by
__global__ void __launch_bounds__(1024) factor_kernel(const float* upstream, int per_token, int64_t tokens, Labels labels, int mean, float unit,
                                                      float* factor, float* back) {
  __shared__ double wide[16];
  __shared__ float narrow[16];
  double count = 0;
  float top = 0.f;
  for (int64_t n = threadIdx.x; n < tokens; n += 1024) {
    const int label = labels.get(n);
    count += label != -1;
    if (label >= 0) top = fmaxf(top, fabsf(upstream[per_token ? n : 0]));
  }
  count = block_reduce(count, [](double a, double b) { return a + b; }, wide);
  top = block_reduce(top, [](float a, float b) { return fmaxf(a, b); }, narrow);
  for (int64_t n = threadIdx.x; n < tokens; n += 1024) {
    const int label = labels.get(n);
    const float g = upstream[per_token ? n : 0];
    factor[n] = label == -1 ? 0.f : label < 0 ? NAN : g == 0.f ? 0.f : g / top;
  }
  if (threadIdx.x == 0) *back = (float)((double)top / (mean ? fmax(count, 1.0) : 1.0) / unit);
}

// E -> G in place; a workgroup per token
template <class T>
__global__ void __launch_bounds__(256) scale_kernel(const Pieces pieces, T* e, const float2* stats, int64_t ld_stats, int64_t token0, Labels labels,
                                                    const float* lse, const float* factor) {
  const int n = blockIdx.x;
  const int64_t ld = (int64_t)pieces.tiles * kTile, at = token0 + n;
  const float log_sum = lse[at], g = factor[at];
  const int label = labels.get(at);
  int64_t want = -1;
  if (label >= 0) {
    int r = 0;
    while (r + 1 < pieces.ranks && label >= pieces.first[r + 1]) ++r;
    want = (int64_t)pieces.tile0[r] * kTile + label - pieces.first[r];
  }
  typedef typename Half<T>::x8 x8;
  for (int64_t v = threadIdx.x * 8; v < ld; v += 256 * 8) {
    const float m = stats[(v >> 7) * ld_stats + n].x;
    const float f = m == -INFINITY ? 0.f : exp_of(m - log_sum) * g;
    x8 o = *(x8*)(e + n * ld + v);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (T)(g == 0.f ? 0.f : (float)o[i] * f - (v + i == want ? kUnit<T> * g : 0.f));
    *(x8*)(e + n * ld + v) = o;
  }
}

// The rows of all ranks' pieces as k of a product, in steps of kStepK; what pads a rank's last tile counts as outside.
struct PieceSource {
  const Pieces* p;
  int64_t stride;
  int col_bytes, r = 0, row = 0;
  __device__ __forceinline__ const char* step(int, int* k_left) {
    while (r + 1 < p->ranks && row >= (p->tile0[r + 1] - p->tile0[r]) * kTile) ++r, row = 0;
    *k_left = min(kStepK, p->rows[r] - row);
    const char* at = *k_left > 0 ? p->w[r] + row * stride + col_bytes : p->w[r];
    row += kStepK;
    return at;
  }
};

struct GradArgs {
  const void* g;     // [tokens][tiles * kTile]
  const char* x;
  int64_t x_stride, w_stride;
  int hidden, tokens, token_tiles, hidden_tiles;
  char* dx;
  int64_t dx_stride, dw_stride;
  const float* back;
  float* sums;       // dw of the pieces so far, [tiles * kTile][hidden]; null: one piece
  int first, last;
};

template <class T>
__global__ void __launch_bounds__(512, 2) dx_kernel(const Pieces pieces, const GradArgs a) {
  typedef TileProduct<T, kTile, kTile, 2, 4, true, false> Product;
  __shared__ __attribute__((aligned(1024))) char smem[Product::kLdsBytes];
  int tt, ht;
  tile_of(blockIdx.x, a.token_tiles, a.hidden_tiles, &tt, &ht);
  const int n0 = tt * kTile, d0 = ht * kTile, tokens = min(kTile, a.tokens - n0), width = min(kTile, a.hidden - d0);
  const int64_t ld = (int64_t)pieces.tiles * kTile;
  f32x4 acc[Product::FL][Product::FR] = {};
  {
    typename Product::LLanes ll;
    typename Product::RLanes rl;
    ll.place(threadIdx.x, a.w_stride, width);
    rl.place(threadIdx.x, ld * 2, tokens);
    Product::run(smem, pieces.tiles * (kTile / kStepK), ll, PieceSource{&pieces, a.w_stride, d0 * 2}, rl, RowSource{(const char*)a.g + n0 * ld * 2, ld}, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l0 = wave % 2 * 128 + (lane >> 4) * 4, r0 = wave / 2 * 64 + (lane & 15);
  const float back = *a.back;
#pragma unroll
  for (int r = 0; r < Product::FR; ++r)
#pragma unroll
    for (int l = 0; l < Product::FL; ++l) {
      const int n = r0 + r * 16, d = l0 + l * 16;
      if (n >= tokens || d >= width) continue;
      typename Half<T>::x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (T)(acc[l][r][i] * back);
      *(typename Half<T>::x4*)(a.dx + (n0 + n) * a.dx_stride + (d0 + d) * 2) = o;
    }
}

template <class T>
__global__ void __launch_bounds__(512, 2) dw_kernel(const Pieces pieces, const Grads grads, const GradArgs a) {
  typedef TileProduct<T, kTile, kTile, 2, 4, true, true> Product;
  __shared__ __attribute__((aligned(1024))) char smem[Product::kLdsBytes];
  int vt, ht;
  tile_of(blockIdx.x, pieces.tiles, a.hidden_tiles, &vt, &ht);
  const int rank = pieces.rank_of(vt), row0 = (vt - pieces.tile0[rank]) * kTile, rows = min(kTile, pieces.rows[rank] - row0);
  const int d0 = ht * kTile, width = min(kTile, a.hidden - d0);
  const int64_t ld = (int64_t)pieces.tiles * kTile;
  f32x4 acc[Product::FL][Product::FR] = {};
  {
    typename Product::LLanes ll;
    typename Product::RLanes rl;
    ll.place(threadIdx.x, a.x_stride, width);
    rl.place(threadIdx.x, ld * 2, kTile);
    Product::run(smem, (a.tokens + kStepK - 1) / kStepK, ll, ColSource{a.x + d0 * 2, a.tokens, a.x_stride}, rl,
                 ColSource{(const char*)a.g + (int64_t)vt * kTile * 2, a.tokens, ld * 2}, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l0 = wave % 2 * 128 + (lane >> 4) * 4, r0 = wave / 2 * 64 + (lane & 15);
  const float back = *a.back;
#pragma unroll
  for (int r = 0; r < Product::FR; ++r)
#pragma unroll
    for (int l = 0; l < Product::FL; ++l) {
      const int v = r0 + r * 16, d = l0 + l * 16;
      if (v >= rows || d >= width) continue;
      f32x4 sum = acc[l][r];
      if (a.sums) {
        f32x4* kept = (f32x4*)(a.sums + ((int64_t)vt * kTile + v) * a.hidden + d0 + d);
        if (!a.first) sum += *kept;
        if (!a.last) {
          *kept = sum;
          continue;
        }
      }
      typename Half<T>::x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (T)(sum[i] * back);
      *(typename Half<T>::x4*)(grads.dw[rank] + (row0 + v) * a.dw_stride + (d0 + d) * 2) = o;
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
  uint64_t off_z = 0, off_loss = 0, off_factor = 0, off_back = 0, off_stats = 0, off_e = 0, off_sums = 0, bytes = 0;
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

struct Call {
  Pieces pieces;
  Grads grads;
  Labels labels;
  float *z_label, *row_loss, *factor, *back, *sums;
  float2* stats;
  void* e;
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
  c->labels = Labels{io->labels, io->label_bytes == 8, d.ignore_index, h->vocab};
  char* ws = (char*)io->workspace;
  c->z_label = (float*)(ws + h->off_z);
  c->row_loss = d.reduction == MSCCLX_LOSS_NONE ? io->loss : (float*)(ws + h->off_loss);
  c->factor = (float*)(ws + h->off_factor);
  c->back = (float*)(ws + h->off_back);
  c->stats = (float2*)(ws + h->off_stats);
  c->e = ws + h->off_e;
  c->sums = h->off_sums ? (float*)(ws + h->off_sums) : nullptr;
  return MSCCLX_OK;
}

int tiles(int64_t n) { return (int)((n + kTile - 1) / kTile); }

template <class T>
int enqueue(const mscclx_vocab_loss* h, const mscclx_vocab_loss_io* io, bool forward, bool backward, const Call& c, hipStream_t stream) {
  const mscclx_vocab_loss_desc& d = h->desc;
  const int64_t n = io->tokens;
  const int mean = d.reduction == MSCCLX_LOSS_MEAN, per_token = d.reduction == MSCCLX_LOSS_NONE;
  int rc;
  if (backward) {
    hipLaunchKernelGGL(factor_kernel, dim3(1), dim3(1024), 0, stream, io->grad_loss, per_token, n, c.labels, mean, kUnit<T>, c.factor, c.back);
    if ((rc = launched("factor_kernel"))) return rc;
  }
  const int hidden_tiles = tiles(d.hidden);
  const int64_t all = std::max<int64_t>(n, backward ? 1 : 0);  // no tokens: dw is still written, with zeros
  for (int64_t at = 0; at < all; at += h->piece) {
    const int now = (int)std::min(h->piece, n - at);
    LogitsArgs a = {};
    a.x = (const char*)io->x + at * io->x_stride * 2;
    a.x_stride = io->x_stride * 2;
    a.w_stride = io->weight_stride * 2;
    a.hidden = d.hidden;
    a.tokens = now;
    a.token_tiles = tiles(now);
    a.token0 = at;
    a.labels = c.labels;
    a.stats = c.stats;
    a.ld_stats = h->piece;
    a.z_label = c.z_label;
    a.e = c.e;
    a.lse = io->lse;
    a.factor = c.factor;
    const dim3 grid((unsigned)(a.token_tiles * c.pieces.tiles));
    if (now > 0) {
      if (!forward) hipLaunchKernelGGL((logits_kernel<T, kGradient>), grid, dim3(512), 0, stream, c.pieces, a);
      else if (backward) hipLaunchKernelGGL((logits_kernel<T, kKeep>), grid, dim3(512), 0, stream, c.pieces, a);
      else hipLaunchKernelGGL((logits_kernel<T, kStats>), grid, dim3(512), 0, stream, c.pieces, a);
      if ((rc = launched("logits_kernel"))) return rc;
      if (forward) {
        hipLaunchKernelGGL(join_kernel, dim3((now + 31) / 32), dim3(256), 0, stream, c.stats, a.ld_stats, 2 * c.pieces.tiles, now, at, c.labels, c.z_label, io->lse, c.row_loss);
        if ((rc = launched("join_kernel"))) return rc;
      }
      if (forward && backward) {
        hipLaunchKernelGGL((scale_kernel<T>), dim3(now), dim3(256), 0, stream, c.pieces, (T*)c.e, c.stats, a.ld_stats, at, c.labels, io->lse, c.factor);
        if ((rc = launched("scale_kernel"))) return rc;
      }
    }
    if (backward) {
      GradArgs g = {};
      g.g = c.e;
      g.x = a.x;
      g.x_stride = a.x_stride;
      g.w_stride = a.w_stride;
      g.hidden = d.hidden;
      g.tokens = now;
      g.token_tiles = a.token_tiles;
      g.hidden_tiles = hidden_tiles;
      g.dx = (char*)io->dx + at * io->dx_stride * 2;
      g.dx_stride = io->dx_stride * 2;
      g.dw_stride = io->dweight_stride * 2;
      g.back = c.back;
      g.sums = n > h->piece ? c.sums : nullptr;
      g.first = at == 0;
      g.last = at + now >= n;
      if (now > 0) {
        hipLaunchKernelGGL((dx_kernel<T>), dim3((unsigned)(g.token_tiles * hidden_tiles)), dim3(512), 0, stream, c.pieces, g);
        if ((rc = launched("dx_kernel"))) return rc;
      }
      hipLaunchKernelGGL((dw_kernel<T>), dim3((unsigned)(c.pieces.tiles * hidden_tiles)), dim3(512), 0, stream, c.pieces, c.grads, g);
      if ((rc = launched("dw_kernel"))) return rc;
    }
  }
  if (forward && d.reduction != MSCCLX_LOSS_NONE) {
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, stream, c.row_loss, n, c.labels, mean, io->loss);
    if ((rc = launched("total_kernel"))) return rc;
  }
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
    for (int r = 0; r < d.ranks; ++r) {
      const int64_t rows = d.rank_rows[r];
      if (rows < 0 || h->vocab + rows > (1ll << 30)) {
        delete h;
        return fail(MSCCLX_ERR_INVALID_ARG, "the ranks' rows must not be negative and add up to at most 2^30");
      }
      p.rows[r] = (int)rows;
      p.first[r] = (int)h->vocab;
      p.tile0[r] = p.tiles;
      p.tiles += tiles(rows);
      h->vocab += rows;
    }
    p.tile0[d.ranks] = p.tiles;
    if (h->vocab == 0) {
      delete h;
      return fail(MSCCLX_ERR_INVALID_ARG, "the vocabulary is empty");
    }
    const uint64_t row = (uint64_t)p.tiles * kTile * 2;  // bytes of E for a token
    const uint64_t budget = d.piece_bytes ? d.piece_bytes : MSCCLX_VOCAB_LOSS_PIECE_BYTES;
    const int64_t fit = (int64_t)(budget / row / kTile * kTile);
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
    h->off_stats = take((uint64_t)h->piece * p.tiles * 2 * sizeof(float2));
    h->off_e = d.gradients ? take((uint64_t)h->piece * row) : 0;
    h->off_sums = d.gradients && d.max_tokens > h->piece ? take((uint64_t)p.tiles * kTile * d.hidden * 4) : 0;
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
