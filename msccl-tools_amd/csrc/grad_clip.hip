// The global norm of the gradients in many tensors, and clipping by it.
//
//   norm = |scale| sqrt(sum g^2)  or  |scale| max |g|      over all tensors that count
//   c    = min(1, max_norm / (norm + 1e-6)),   out = g scale c
//
// Tensors are cut into chunks; a table in the workspace holds each chunk's addresses, so that a workgroup is two
// dependent loads from its data.  Workgroup b takes chunks b, b + grid, ...
//
// The first kernel reads every counted chunk once: squares are added in 64 bits (they are exact there, so no large
// gradient overflows and no small one is lost; two conversions and a multiply-add per element, a fifth of what memory
// takes), magnitudes are compared as unsigned integers, in which NaN is above infinity.  Each workgroup leaves one
// partial result.  The norm alone: the last workgroup to arrive adds the partial results, in one order.  Clipping: a
// second kernel, in which every workgroup adds them, in the same order, and scales its chunks.  No sum goes through an
// atomic: the same bits at every call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <string>
#include <memory>
#include <type_traits>
#include <vector>

#include "plan.h"

namespace mscclx {
namespace {

constexpr int kMinChunk = 2048, kMaxChunk = 16384;  // elements
constexpr int kMaxGrid = 2048;                         // workgroups, and partial results
constexpr int kThreads = 256;
constexpr int kArrivals = 64;                          // counters of finished workgroups: one for all is a queue of 2048

struct Chunk {
  const void* in;
  void* out;
  uint32_t n;
  uint8_t in_type, out_type, counted, reserved[9];
};
static_assert(sizeof(Chunk) == 32, "two 16-byte loads");

struct alignas(256) Header {
  float norm, coefficient;
  unsigned done;                  // counters whose last workgroup has arrived
  unsigned arrived[kArrivals][16];  // each alone in 64 bytes; the last to arrive leaves zeros
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }
__device__ __forceinline__ float widen(__bf16 x) { return (float)x; }

// elements in any alignment of their type: the hardware takes 16-byte accesses on every boundary
template <class T, int N> __device__ __forceinline__ void load(const T* p, T (&out)[N]) { __builtin_memcpy(out, p, sizeof(out)); }
template <class T, int N> __device__ __forceinline__ void store(T* p, const T (&in)[N]) { __builtin_memcpy(p, in, sizeof(in)); }

template <class F> __device__ __forceinline__ void by_type(int type, F f) {
  switch (type) {
    case MSCCLX_F32: f((float*)nullptr); break;
    case MSCCLX_BF16: f((__bf16*)nullptr); break;
    default: f((_Float16*)nullptr); break;
  }
}

template <class V, class F> __device__ __forceinline__ V over_workgroup(V v, F f, V* shared) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = f(v, __shfl_xor(v, d));
  if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
  __syncthreads();
  v = shared[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v = f(v, shared[w]);
  __syncthreads();
  return v;
}

// One accumulator for both norms: squares in 64 bits, or the magnitude's bits.
template <bool MAX> struct Norm;
template <> struct Norm<false> {
  typedef double value;
  static __device__ __forceinline__ double of(double a, float x) { return a + (double)x * (double)x; }
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
  static __device__ __forceinline__ double result(double a) { return sqrt(a); }
};
template <> struct Norm<true> {
  typedef unsigned value;
  static __device__ __forceinline__ unsigned of(unsigned a, float x) { return max(a, __float_as_uint(x) & 0x7fffffffu); }
  static __device__ __forceinline__ unsigned join(unsigned a, unsigned b) { return max(a, b); }
  static __device__ __forceinline__ double result(unsigned a) { return (double)__uint_as_float(a); }
};

// The result from the partial results' sum; `threadIdx.x == 0` writes it.  Returns the factor, in 64 bits: against gradients
// of 1e36 it is below what 32 bits hold, and the output is nevertheless an ordinary number.
template <bool MAX>
__device__ __forceinline__ double finish(typename Norm<MAX>::value sum, double scale, double max_norm, Header* header, bool writes) {
  const double norm = Norm<MAX>::result(sum) * fabs(scale);
  double c = 1.0;
  if (max_norm >= 0.0) {
    c = max_norm / (norm + 1e-6);
    if (c >= 1.0) c = 1.0;  // (a NaN stays)
  }
  if (writes && threadIdx.x == 0) {
    header->norm = (float)norm;
    header->coefficient = (float)c;
  }
  return c * scale;
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_kernel(const Chunk* chunks, int nchunks, typename Norm<MAX>::value* partial, int alone, double scale, Header* header) {
  typedef Norm<MAX> N;
  typedef typename N::value V;
  __shared__ V shared[kThreads / 64];
  V sum = 0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const Chunk t = chunks[c];
    if (!t.counted) continue;
    by_type(t.in_type, [&](auto* type) {
      typedef std::remove_pointer_t<decltype(type)> T;
      constexpr int W = 16 / sizeof(T);
      const T* p = (const T*)t.in;
      const int n = (int)t.n;
      int i = threadIdx.x * W;
#pragma unroll 4
      for (; i + W <= n; i += kThreads * W) {
        T v[W];
        load(p + i, v);
#pragma unroll
        for (int k = 0; k < W; ++k) sum = N::of(sum, widen(v[k]));
      }
      for (; i < n && i + W > n; ++i) sum = N::of(sum, widen(p[i]));  // the one thread at the end
    });
  }
  auto join = [](V a, V b) { return N::join(a, b); };
  sum = over_workgroup(sum, join, shared);
  if (!alone) {
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
    return;
  }
  // Who arrives last adds: of the workgroups of a counter, then of the counters.  Release and acquire would write back
  // and drop this XCD's cache for every workgroup (norm over 256 MiB: 101 us instead of 42).  They are not needed: the
  // partial result is exchanged, not stored, so its old value comes back only when the new one is where all XCDs see
  // it, and each next atomic waits for the value of the one before; the loads below go to the same place.
  __shared__ int last;
  if (threadIdx.x == 0) {
    typedef std::conditional_t<sizeof(V) == 8, unsigned long long, unsigned> Bits;
    const Bits before = __hip_atomic_exchange((Bits*)&partial[blockIdx.x], __builtin_bit_cast(Bits, sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::"v"(before) : "memory");
    const unsigned grid = gridDim.x, mine = blockIdx.x % kArrivals, of_mine = (grid - mine + kArrivals - 1) / kArrivals;
    last = 0;
    if (__hip_atomic_fetch_add(&header->arrived[mine][0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == of_mine) {
      __hip_atomic_store(&header->arrived[mine][0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (__hip_atomic_fetch_add(&header->done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == min(grid, (unsigned)kArrivals)) {
        __hip_atomic_store(&header->done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = 1;
      }
    }
  }
  __syncthreads();
  if (!last) return;
  sum = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kThreads) sum = N::join(sum, __hip_atomic_load(&partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  finish<MAX>(over_workgroup(sum, join, shared), scale, -1.0, header, true);
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) scale_kernel(const Chunk* chunks, int nchunks, const typename Norm<MAX>::value* partial, double scale, double max_norm,
                                                         Header* header) {
  typedef Norm<MAX> N;
  typedef typename N::value V;
  __shared__ V shared[kThreads / 64];
  V sum = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kThreads) sum = N::join(sum, partial[i]);
  const double factor = finish<MAX>(over_workgroup(sum, [](V a, V b) { return N::join(a, b); }, shared), scale, max_norm, header, blockIdx.x == 0);
  for (int b = blockIdx.x; b < nchunks; b += gridDim.x) {
    const Chunk t = chunks[b];
    if (factor == 1.0 && t.in == t.out) continue;  // nothing changes (in place, types are the same)
    by_type(t.in_type, [&](auto* in_type) {
      by_type(t.out_type, [&](auto* out_type) {
        typedef std::remove_pointer_t<decltype(in_type)> T;
        typedef std::remove_pointer_t<decltype(out_type)> U;
        constexpr int W = 16 / std::max(sizeof(T), sizeof(U));
        const T* p = (const T*)t.in;
        U* q = (U*)t.out;
        const int n = (int)t.n;
        int i = threadIdx.x * W;
#pragma unroll 4
        for (; i + W <= n; i += kThreads * W) {
          T v[W];
          U o[W];
          load(p + i, v);
#pragma unroll
          for (int k = 0; k < W; ++k) o[k] = (U)(float)(widen(v[k]) * factor);
          store(q + i, o);
        }
        for (; i < n && i + W > n; ++i) q[i] = (U)(float)(widen(p[i]) * factor);
      });
    });
  }
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSCCLX_OK : fail(MSCCLX_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

template <class F> int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return MSCCLX_ERR_CAPACITY;
  } catch (...) {
    return MSCCLX_ERR_INVALID_ARG;
  }
}

}  // namespace
}  // namespace mscclx

using namespace mscclx;

struct mscclx_grad_clip {
  struct Tensor {
    uint64_t n;
    int32_t in_type, out_type;
    bool counted;
  };
  std::vector<Tensor> tensors;
  int norm = 0;
  uint64_t chunk = kMinChunk;  // elements
  uint64_t chunks = 0;
  uint64_t off_partial = 0, off_chunks = 0, bytes = 0;
  char* workspace = nullptr;  // of the last bind
  bool outputs = false;
};

extern "C" {

int mscclx_grad_clip_create(int32_t ntensors, const uint64_t* sizes, const int32_t* in_dtypes, const int32_t* out_dtypes, const uint8_t* counted,
                            int32_t norm, mscclx_grad_clip** out, uint64_t* workspace_bytes) {
  return guarded([&] {
    if (!out || ntensors < 0 || (ntensors && (!sizes || !in_dtypes || !out_dtypes))) return fail(MSCCLX_ERR_INVALID_ARG, "null argument");
    *out = nullptr;
    if (norm != MSCCLX_NORM_L2 && norm != MSCCLX_NORM_MAX) return fail(MSCCLX_ERR_INVALID_ARG, "unknown norm");
    auto type_ok = [](int32_t t) { return t == MSCCLX_F32 || t == MSCCLX_F16 || t == MSCCLX_BF16; };
    std::unique_ptr<mscclx_grad_clip> h(new mscclx_grad_clip());
    h->norm = norm;
    uint64_t total = 0;
    for (int i = 0; i < ntensors; ++i) {
      if (!type_ok(in_dtypes[i]) || !type_ok(out_dtypes[i]))
        return fail(MSCCLX_ERR_UNSUPPORTED, "tensor " + std::to_string(i) + ": gradients are float32, float16 or bfloat16");
      if (sizes[i] > (1ull << 40)) return fail(MSCCLX_ERR_INVALID_ARG, "tensor " + std::to_string(i) + ": more than 2^40 elements");
      total += sizes[i];
      if (total > (1ull << 44)) return fail(MSCCLX_ERR_CAPACITY, "more than 2^44 gradients");
      h->tensors.push_back({sizes[i], in_dtypes[i], out_dtypes[i], !counted || counted[i]});
    }
    // eight chunks for each workgroup of a full grid, so that the last ones are short against the whole; of at least
    // one pass of its threads
    while (h->chunk < kMaxChunk && h->chunk * kMaxGrid * 8 < total) h->chunk *= 2;
    for (const auto& t : h->tensors) h->chunks += (t.n + h->chunk - 1) / h->chunk;
    uint64_t at = (sizeof(Header) + 255) / 256 * 256;
    auto take = [&](uint64_t bytes) {
      const uint64_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    h->off_partial = take(kMaxGrid * sizeof(double));
    h->off_chunks = take(h->chunks * sizeof(Chunk));
    h->bytes = at;
    if (workspace_bytes) *workspace_bytes = at;
    *out = h.release();
    return (int)MSCCLX_OK;
  });
}

int mscclx_grad_clip_destroy(mscclx_grad_clip* clip) {
  delete clip;
  return MSCCLX_OK;
}

int mscclx_grad_clip_bind(mscclx_grad_clip* h, const void* const* in, void* const* out, void* workspace, uint64_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (!h) return fail(MSCCLX_ERR_INVALID_ARG, "null argument");
    if (workspace_bytes < h->bytes)
      return fail(MSCCLX_ERR_CAPACITY, "workspace of " + std::to_string(workspace_bytes) + " bytes given, " + std::to_string(h->bytes) + " needed");
    if (!workspace || (uintptr_t)workspace % 256) return fail(MSCCLX_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
    struct Span {
      uintptr_t from, to;
      int tensor;
      bool written;
    };
    std::vector<Span> spans;
    std::vector<Chunk> chunks;
    chunks.reserve(h->chunks);
    for (size_t i = 0; i < h->tensors.size(); ++i) {
      const mscclx_grad_clip::Tensor& t = h->tensors[i];
      if (!t.n) continue;
      const std::string name = "tensor " + std::to_string(i);
      const uintptr_t a = in ? (uintptr_t)in[i] : 0, b = out ? (uintptr_t)out[i] : 0;
      if (!a || (out && !b)) return fail(MSCCLX_ERR_INVALID_ARG, name + ": NULL");
      const uint64_t in_size = dtype_size(t.in_type), out_size = dtype_size(t.out_type);
      if (a % in_size || b % out_size) return fail(MSCCLX_ERR_INVALID_ARG, name + ": not aligned to its element type");
      const bool in_place = out && a == b;
      if (in_place && t.in_type != t.out_type) return fail(MSCCLX_ERR_ALIASED, name + ": in place, but its types differ");
      spans.push_back({a, a + t.n * in_size, (int)i, in_place});
      if (out && !in_place) spans.push_back({b, b + t.n * out_size, (int)i, true});
      for (uint64_t from = 0; from < t.n; from += h->chunk)
        chunks.push_back({(const void*)(a + from * in_size), out ? (void*)(b + from * out_size) : nullptr, (uint32_t)std::min(h->chunk, t.n - from), (uint8_t)t.in_type,
                          (uint8_t)t.out_type, (uint8_t)t.counted, {}});
    }
    spans.push_back({(uintptr_t)workspace, (uintptr_t)workspace + h->bytes, -1, true});
    // what one tensor writes, and the workspace, no other may read or write (two inputs may share memory)
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    uintptr_t read_to = 0, written_to = 0;
    for (const Span& s : spans) {
      if (s.from < written_to || (s.written && s.from < read_to))
        return fail(MSCCLX_ERR_ALIASED, (s.tensor < 0 ? "the workspace" : "tensor " + std::to_string(s.tensor)) + ": its memory overlaps another buffer, one of them written");
      (s.written ? written_to : read_to) = std::max(s.written ? written_to : read_to, s.to);
    }
    char* ws = (char*)workspace;
    hipStream_t s = (hipStream_t)stream;
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &capturing) != hipSuccess || capturing != hipStreamCaptureStatusNone) {
      (void)hipGetLastError();
      return fail(MSCCLX_ERR_STATE, "tensors are bound before a stream is captured, not meanwhile");
    }
    h->workspace = nullptr;  // (until the new table is there)
    const Header zeros = {};
    hipError_t e = hipMemcpyAsync(ws, &zeros, sizeof(Header), hipMemcpyHostToDevice, s);
    if (e == hipSuccess && !chunks.empty()) e = hipMemcpyAsync(ws + h->off_chunks, chunks.data(), chunks.size() * sizeof(Chunk), hipMemcpyHostToDevice, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) return fail(MSCCLX_ERR_HIP, std::string("uploading the table of gradients: ") + hipGetErrorString(e));
    h->workspace = ws;
    h->outputs = out != nullptr;
    return (int)MSCCLX_OK;
  });
}

int mscclx_grad_clip_launch(const mscclx_grad_clip* h, double scale, double max_norm, void* stream) {
  return guarded([&] {
    if (!h || !h->workspace) return fail(MSCCLX_ERR_STATE, "bind tensors before launching");
    if (!std::isfinite(scale)) return fail(MSCCLX_ERR_INVALID_ARG, "scale must be finite");
    if (std::isnan(max_norm)) return fail(MSCCLX_ERR_INVALID_ARG, "max_norm must be a number");
    const bool clip = max_norm >= 0.0;
    if (clip && !h->outputs) return fail(MSCCLX_ERR_STATE, "the tensors were bound without outputs");
    char* ws = h->workspace;
    const int nchunks = (int)h->chunks, grid = std::max(1, std::min(nchunks, kMaxGrid));
    const Chunk* chunks = (const Chunk*)(ws + h->off_chunks);
    Header* header = (Header*)ws;
    hipStream_t s = (hipStream_t)stream;
    auto both = [&](auto max) -> int {
      constexpr bool MAX = decltype(max)::value;
      auto* partial = (typename Norm<MAX>::value*)(ws + h->off_partial);
      hipLaunchKernelGGL((norm_kernel<MAX>), dim3(grid), dim3(kThreads), 0, s, chunks, nchunks, partial, (int)!clip, scale, header);
      if (int rc = launched("norm_kernel")) return rc;
      if (!clip) return MSCCLX_OK;
      hipLaunchKernelGGL((scale_kernel<MAX>), dim3(grid), dim3(kThreads), 0, s, chunks, nchunks, partial, scale, max_norm, header);
      return launched("scale_kernel");
    };
    return h->norm == MSCCLX_NORM_MAX ? both(std::true_type()) : both(std::false_type());
  });
}

}  // extern "C"
