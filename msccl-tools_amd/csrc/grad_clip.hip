// The global norm of the gradients in many tensors, and clipping by it.
//
//   norm = |scale| sqrt(sum g^2)  or  |scale| max |g|      over all tensors that count
//   c    = min(1, max_norm / (norm + 1e-6)),   out = g scale c
//
// Two launches.  The first reads every counted tensor once: squares are added in 64 bits (exact for the squares themselves, so no large
// gradient overflows and no small one is lost; two conversions' and one multiply-add's time per element, a fifth of what memory takes), magnitudes are compared as
// unsigned integers, in which NaN is above infinity.  Each workgroup leaves one partial result.  The second adds the partial
// results in one order in every workgroup (no atomics: the same bits at every call) and scales.  Tensors are cut
// into chunks of kChunk elements; workgroup b takes chunks b, b + grid, ...  The second launch walks them backwards: what the first read last
// is still in the memory-side cache.
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

constexpr int kChunk = 16384;    // elements
constexpr int kMaxGrid = 2048;   // workgroups, and partial results
constexpr int kThreads = 256;

struct Tensor {
  const void* in;
  void* out;
  uint64_t n;
  int32_t in_type, out_type;
  int32_t counted, reserved;
};
struct Chunk {
  uint32_t tensor, index;
};

struct alignas(256) Header {
  float norm, coefficient;
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

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_kernel(const Tensor* tensors, const Chunk* chunks, int nchunks, typename Norm<MAX>::value* partial) {
  typedef Norm<MAX> N;
  __shared__ typename N::value shared[kThreads / 64];
  typename N::value sum = 0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const Chunk chunk = chunks[c];
    const Tensor t = tensors[chunk.tensor];
    if (!t.counted) continue;
    const uint64_t from = (uint64_t)chunk.index * kChunk;
    const int n = (int)min((uint64_t)kChunk, t.n - from);
    by_type(t.in_type, [&](auto* type) {
      typedef std::remove_pointer_t<decltype(type)> T;
      constexpr int W = 16 / sizeof(T);
      const T* p = (const T*)t.in + from;
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
  sum = over_workgroup(sum, [](auto a, auto b) { return N::join(a, b); }, shared);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// the partial results' sum in every workgroup, in the same order
template <bool MAX>
__device__ __forceinline__ float factor_of(const typename Norm<MAX>::value* partial, int count, float scale, float max_norm, Header* header) {
  typedef Norm<MAX> N;
  __shared__ typename N::value shared[kThreads / 64];
  typename N::value sum = 0;
  for (int i = threadIdx.x; i < count; i += kThreads) sum = N::join(sum, partial[i]);
  sum = over_workgroup(sum, [](auto a, auto b) { return N::join(a, b); }, shared);
  const double norm = N::result(sum) * fabs((double)scale);
  double c = 1.0;
  if (max_norm >= 0.f) {
    c = (double)max_norm / (norm + 1e-6);
    if (c >= 1.0) c = 1.0;  // (a NaN stays)
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    header->norm = (float)norm;
    header->coefficient = (float)c;
  }
  return (float)(c * scale);
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) finish_kernel(const typename Norm<MAX>::value* partial, int count, float scale, Header* header) {
  factor_of<MAX>(partial, count, scale, -1.f, header);
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) scale_kernel(const Tensor* tensors, const Chunk* chunks, int nchunks, const typename Norm<MAX>::value* partial,
                                                         int count, float scale, float max_norm, Header* header) {
  const float factor = factor_of<MAX>(partial, count, scale, max_norm, header);
  for (int b = blockIdx.x; b < nchunks; b += gridDim.x) {
    const Chunk chunk = chunks[nchunks - 1 - b];
    const Tensor t = tensors[chunk.tensor];
    if (factor == 1.f && t.in == t.out) continue;  // nothing changes (in place, types are the same)
    const uint64_t from = (uint64_t)chunk.index * kChunk;
    const int n = (int)min((uint64_t)kChunk, t.n - from);
    by_type(t.in_type, [&](auto* in_type) {
      by_type(t.out_type, [&](auto* out_type) {
        typedef std::remove_pointer_t<decltype(in_type)> T;
        typedef std::remove_pointer_t<decltype(out_type)> U;
        constexpr int W = 16 / sizeof(T);
        const T* p = (const T*)t.in + from;
        U* q = (U*)t.out + from;
        int i = threadIdx.x * W;
#pragma unroll 4
        for (; i + W <= n; i += kThreads * W) {
          T v[W];
          U o[W];
          load(p + i, v);
#pragma unroll
          for (int k = 0; k < W; ++k) o[k] = (U)(widen(v[k]) * factor);
          store(q + i, o);
        }
        for (; i < n && i + W > n; ++i) q[i] = (U)(widen(p[i]) * factor);
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
  std::vector<Tensor> tensors;
  std::vector<Chunk> chunks;
  int norm = 0;
  uint64_t off_partial = 0, off_tensors = 0, off_chunks = 0, bytes = 0;
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
    uint64_t chunks = 0;
    for (int i = 0; i < ntensors; ++i) {
      if (!type_ok(in_dtypes[i]) || !type_ok(out_dtypes[i]))
        return fail(MSCCLX_ERR_UNSUPPORTED, "tensor " + std::to_string(i) + ": gradients are float32, float16 or bfloat16");
      if (sizes[i] > (1ull << 40)) return fail(MSCCLX_ERR_INVALID_ARG, "tensor " + std::to_string(i) + ": more than 2^40 elements");
      chunks += (sizes[i] + kChunk - 1) / kChunk;
      if (chunks > (1ull << 30)) return fail(MSCCLX_ERR_CAPACITY, "more than 2^30 chunks of gradients");
    }
    h->tensors.reserve(ntensors);
    h->chunks.reserve(chunks);
    for (int i = 0; i < ntensors; ++i) {
      h->tensors.push_back(Tensor{nullptr, nullptr, sizes[i], in_dtypes[i], out_dtypes[i], counted ? counted[i] != 0 : 1, 0});
      for (uint64_t c = 0; c < (sizes[i] + kChunk - 1) / kChunk; ++c) h->chunks.push_back(Chunk{(uint32_t)i, (uint32_t)c});
    }
    uint64_t at = sizeof(Header);
    auto take = [&](uint64_t bytes) {
      const uint64_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    h->off_partial = take(kMaxGrid * sizeof(double));
    h->off_tensors = take(h->tensors.size() * sizeof(Tensor));
    h->off_chunks = take(h->chunks.size() * sizeof(Chunk));
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
    std::vector<Tensor> tensors = h->tensors;
    for (size_t i = 0; i < tensors.size(); ++i) {
      Tensor& t = tensors[i];
      t.in = t.n && in ? in[i] : nullptr;
      t.out = t.n && out ? out[i] : nullptr;
      if (!t.n) continue;
      const std::string name = "tensor " + std::to_string(i);
      if (!t.in || (out && !t.out)) return fail(MSCCLX_ERR_INVALID_ARG, name + ": NULL");
      const uintptr_t in_size = dtype_size(t.in_type), out_size = dtype_size(t.out_type);
      if ((uintptr_t)t.in % in_size || (uintptr_t)t.out % out_size) return fail(MSCCLX_ERR_INVALID_ARG, name + ": not aligned to its element type");
      if (out && t.in == t.out && t.in_type != t.out_type) return fail(MSCCLX_ERR_ALIASED, name + ": in place, but its types differ");
      const uintptr_t a = (uintptr_t)t.in, b = (uintptr_t)t.out;
      const bool in_place = out && a == b;
      spans.push_back({a, a + t.n * in_size, (int)i, in_place});
      if (out && !in_place) spans.push_back({b, b + t.n * out_size, (int)i, true});
    }
    // what one tensor writes no other may read or write (two inputs may share memory)
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    uintptr_t read_to = 0, written_to = 0;
    for (const Span& s : spans) {
      if (s.from < written_to || (s.written && s.from < read_to)) return fail(MSCCLX_ERR_ALIASED, "tensor " + std::to_string(s.tensor) + ": its memory overlaps another buffer, one of them an output");
      (s.written ? written_to : read_to) = std::max(s.written ? written_to : read_to, s.to);
    }
    char* ws = (char*)workspace;
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    if (!tensors.empty()) e = hipMemcpyAsync(ws + h->off_tensors, tensors.data(), tensors.size() * sizeof(Tensor), hipMemcpyHostToDevice, s);
    if (e == hipSuccess && !h->chunks.empty()) e = hipMemcpyAsync(ws + h->off_chunks, h->chunks.data(), h->chunks.size() * sizeof(Chunk), hipMemcpyHostToDevice, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) {
      h->workspace = nullptr;
      return fail(MSCCLX_ERR_HIP, std::string("uploading the table of tensors: ") + hipGetErrorString(e));
    }
    h->workspace = ws;
    h->outputs = out != nullptr;
    return (int)MSCCLX_OK;
  });
}

int mscclx_grad_clip_launch(const mscclx_grad_clip* h, float scale, float max_norm, void* stream) {
  return guarded([&] {
    if (!h || !h->workspace) return fail(MSCCLX_ERR_STATE, "bind tensors before launching");
    if (!std::isfinite(scale)) return fail(MSCCLX_ERR_INVALID_ARG, "scale must be finite");
    if (std::isnan(max_norm)) return fail(MSCCLX_ERR_INVALID_ARG, "max_norm must be a number");
    const bool clip = max_norm >= 0.f;
    if (clip && !h->outputs) return fail(MSCCLX_ERR_STATE, "the tensors were bound without outputs");
    char* ws = h->workspace;
    const int nchunks = (int)h->chunks.size(), grid = std::max(1, std::min(nchunks, kMaxGrid));
    const Tensor* tensors = (const Tensor*)(ws + h->off_tensors);
    const Chunk* chunks = (const Chunk*)(ws + h->off_chunks);
    hipStream_t s = (hipStream_t)stream;
    auto both = [&](auto max) -> int {
      constexpr bool MAX = decltype(max)::value;
      auto* partial = (typename Norm<MAX>::value*)(ws + h->off_partial);
      hipLaunchKernelGGL((norm_kernel<MAX>), dim3(grid), dim3(kThreads), 0, s, tensors, chunks, nchunks, partial);
      if (int rc = launched("norm_kernel")) return rc;
      if (!clip) hipLaunchKernelGGL((finish_kernel<MAX>), dim3(1), dim3(kThreads), 0, s, partial, grid, scale, (Header*)ws);
      else hipLaunchKernelGGL((scale_kernel<MAX>), dim3(grid), dim3(kThreads), 0, s, tensors, chunks, nchunks, partial, grid, scale, max_norm, (Header*)ws);
      return launched(clip ? "scale_kernel" : "finish_kernel");
    };
    return h->norm == MSCCLX_NORM_MAX ? both(std::true_type()) : both(std::false_type());
  });
}

}  // extern "C"
