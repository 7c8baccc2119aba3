// The 2-norm over every element of a list of tensors, and clipping the list by it.
//
//   norm = sqrt(sum_t sum_i g_t[i]^2);   out_t[i] = g_t[i] min(1, max_norm / (norm + 1e-6))
//
// The list travels in the launch's parameters (no copy to the device, so a captured call replays as it is).  Every
// tensor is cut into chunks of kChunk elements and the chunks of the list are dealt to the blocks in equal runs, so a
// list of many small tensors and one of few large ones load the GPU alike.  Squares and sums are fp64: a square of any
// finite fp32 value neither overflows nor vanishes, and the sum's order is fixed (no atomics).
#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include <cuda_fp16.h>

#include "bpc.h"
#include "bpc_common.cuh"
#include "bpc_internal.h"

namespace bpc {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;              // elements
constexpr int kListMax = 1000;            // tensors per launch: 32 bytes each, within the 32,764 bytes of parameters
constexpr int kBlocksPerSm = 8;

struct Entry {
  const void* in;
  void* out;
  int64_t numel;
  int32_t first_chunk;                    // chunks of the list before this tensor
  int16_t in_dtype, out_dtype;
};

template <int N>
struct List {
  int32_t n, chunks;
  Entry e[N];
};

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// the last entry whose chunks begin at or before chunk k
template <int N>
__device__ __forceinline__ int find_entry(const List<N>& list, int k) {
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.e[mid].first_chunk <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// the sum over the block, in every thread; red: kThreads / 32 doubles
__device__ __forceinline__ double block_sum(double v, double* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}

// elements before the first 16-byte boundary at or after p
template <typename T>
__device__ __forceinline__ int peel_of(const T* p, int len) {
  const int k = static_cast<int>(((0 - reinterpret_cast<uintptr_t>(p)) & 15) / sizeof(T));
  return k < len ? k : len;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* __restrict__ p, int len) {
  constexpr int VEC = 16 / sizeof(T);
  const int peel = peel_of(p, len);
  const int nv = (len - peel) / VEC;
  double s = 0.0;
  if (static_cast<int>(threadIdx.x) < peel) {
    const double x = load_f32(p + threadIdx.x);
    s = x * x;
  }
  const Pack<T, VEC>* v = reinterpret_cast<const Pack<T, VEC>*>(p + peel);
#pragma unroll 4
  for (int i = threadIdx.x; i < nv; i += kThreads) {
    const Pack<T, VEC> x = v[i];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const double d = load_f32(&x.v[e]);
      s = fma(d, d, s);
    }
  }
  const int t = peel + nv * VEC + threadIdx.x;
  if (t < len) {
    const double x = load_f32(p + t);
    s = fma(x, x, s);
  }
  return s;
}

template <int N>
__global__ void __launch_bounds__(kThreads) norm_partial_kernel(const __grid_constant__ List<N> list, int per_block,
                                                                double* __restrict__ partial) {
  __shared__ double red[kThreads / 32];
  const int k0 = blockIdx.x * per_block, k1 = min(list.chunks, k0 + per_block);
  double s = 0.0;
  int t = k0 < k1 ? find_entry(list, k0) : 0;
  for (int k = k0; k < k1; ++k) {
    while (t + 1 < list.n && list.e[t + 1].first_chunk <= k) ++t;
    const Entry& e = list.e[t];
    const int64_t off = static_cast<int64_t>(k - e.first_chunk) * kChunk;
    const int len = static_cast<int>(min(static_cast<int64_t>(kChunk), e.numel - off));
    if (e.in_dtype == BPC_DTYPE_F32) s += chunk_squares(static_cast<const float*>(e.in) + off, len);
    else if (e.in_dtype == BPC_DTYPE_BF16) s += chunk_squares(static_cast<const __nv_bfloat16*>(e.in) + off, len);
    else s += chunk_squares(static_cast<const __half*>(e.in) + off, len);
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// the sum of the blocks' partial sums, the same in every thread and block
__device__ __forceinline__ double total_squares(const double* __restrict__ partial, int partials, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) s += partial[i];
  return block_sum(s, red);
}

__global__ void __launch_bounds__(kThreads) norm_finish_kernel(const double* __restrict__ partial, int partials,
                                                               float* __restrict__ norm) {
  __shared__ double red[kThreads / 32];
  const double s = total_squares(partial, partials, red);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(s));
}

template <typename T, typename U>
__device__ __forceinline__ void chunk_scale(const T* p, U* q, int len, double coef) {
  constexpr int VEC = 16 / sizeof(T);
  const float c = static_cast<float>(coef);
  // a factor below fp32's normal range (a norm beyond 1e37) would lose bits: multiply in fp64 then
  const bool tiny = coef < 1.1754944e-38;
  auto scaled = [&](float x) { return tiny ? static_cast<float>(x * coef) : x * c; };
  const int peel = peel_of(p, len);
  const int nv = (len - peel) / VEC;
  if (static_cast<int>(threadIdx.x) < peel) store_f32(q + threadIdx.x, scaled(load_f32(p + threadIdx.x)));
  const Pack<T, VEC>* v = reinterpret_cast<const Pack<T, VEC>*>(p + peel);
  U* o = q + peel;
  constexpr int OVEC = sizeof(U) * VEC > 16 ? 16 / sizeof(U) : VEC;       // elements per store
  const bool wide = reinterpret_cast<uintptr_t>(o) % (sizeof(U) * OVEC) == 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < nv; i += kThreads) {
    const Pack<T, VEC> x = v[i];
    Pack<U, VEC> y;
#pragma unroll
    for (int e = 0; e < VEC; ++e) store_f32(&y.v[e], scaled(load_f32(&x.v[e])));
    if (wide) {
#pragma unroll
      for (int e = 0; e < VEC; e += OVEC)
        *reinterpret_cast<Pack<U, OVEC>*>(o + static_cast<int64_t>(i) * VEC + e) =
            *reinterpret_cast<const Pack<U, OVEC>*>(&y.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[static_cast<int64_t>(i) * VEC + e] = y.v[e];
    }
  }
  const int t = peel + nv * VEC + threadIdx.x;
  if (t < len) store_f32(q + t, scaled(load_f32(p + t)));
}

template <typename T>
__device__ __forceinline__ void chunk_scale_to(const T* p, void* out, int dtype, int64_t off, int len, double coef) {
  if (dtype == BPC_DTYPE_F32) chunk_scale(p + off, static_cast<float*>(out) + off, len, coef);
  else if (dtype == BPC_DTYPE_BF16) chunk_scale(p + off, static_cast<__nv_bfloat16*>(out) + off, len, coef);
  else chunk_scale(p + off, static_cast<__half*>(out) + off, len, coef);
}

template <int N>
__global__ void __launch_bounds__(kThreads) clip_scale_kernel(const __grid_constant__ List<N> list, int per_block,
                                                              const double* __restrict__ partial, int partials,
                                                              double max_norm, float* __restrict__ norm) {
  __shared__ double red[kThreads / 32];
  const double total = sqrt(total_squares(partial, partials, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
  double coef = max_norm / (total + 1e-6);
  if (coef > 1.0) coef = 1.0;             // a NaN stays
  const int k0 = blockIdx.x * per_block, k1 = min(list.chunks, k0 + per_block);
  int t = k0 < k1 ? find_entry(list, k0) : 0;
  for (int k = k0; k < k1; ++k) {
    while (t + 1 < list.n && list.e[t + 1].first_chunk <= k) ++t;
    const Entry& e = list.e[t];
    if (coef == 1.0 && e.in == e.out) continue;           // in place and within the limit: nothing changes
    const int64_t off = static_cast<int64_t>(k - e.first_chunk) * kChunk;
    const int len = static_cast<int>(min(static_cast<int64_t>(kChunk), e.numel - off));
    if (e.in_dtype == BPC_DTYPE_F32)
      chunk_scale_to(static_cast<const float*>(e.in), e.out, e.out_dtype, off, len, coef);
    else if (e.in_dtype == BPC_DTYPE_BF16)
      chunk_scale_to(static_cast<const __nv_bfloat16*>(e.in), e.out, e.out_dtype, off, len, coef);
    else
      chunk_scale_to(static_cast<const __half*>(e.in), e.out, e.out_dtype, off, len, coef);
  }
}

int size_of(int32_t dtype) { return dtype == BPC_DTYPE_F32 ? 4 : dtype == BPC_DTYPE_BF16 || dtype == BPC_DTYPE_F16 ? 2 : 0; }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

int max_blocks() { return kBlocksPerSm * num_sms(); }
int launches_of(int32_t n) { return (n + kListMax - 1) / kListMax; }

// One launch's share of the list: tensors [t0, t1)
struct Part {
  int t0, t1, chunks, per_block, blocks;
};

std::vector<Part> parts_of(const int64_t* numel, int32_t n) {
  std::vector<Part> parts;
  for (int t0 = 0; t0 < n; t0 += kListMax) {
    Part p{t0, std::min(n, t0 + kListMax), 0, 1, 0};
    int64_t chunks = 0;
    for (int t = p.t0; t < p.t1; ++t) chunks += (numel[t] + kChunk - 1) / kChunk;
    p.chunks = static_cast<int>(chunks);
    p.per_block = std::max(1, (p.chunks + max_blocks() - 1) / max_blocks());
    p.blocks = (p.chunks + p.per_block - 1) / p.per_block;
    parts.push_back(p);
  }
  return parts;
}

template <int N>
void fill(List<N>* list, const Part& p, const void* const* in, void* const* out, const int64_t* numel,
          const int32_t* in_dtype, const int32_t* out_dtype) {
  list->n = 0;
  list->chunks = p.chunks;
  int chunk = 0;
  for (int t = p.t0; t < p.t1; ++t) {
    if (numel[t] == 0) continue;
    Entry& e = list->e[list->n++];
    e.in = in[t];
    e.out = out ? out[t] : nullptr;
    e.numel = numel[t];
    e.first_chunk = chunk;
    e.in_dtype = static_cast<int16_t>(in_dtype[t]);
    e.out_dtype = static_cast<int16_t>(out_dtype ? out_dtype[t] : in_dtype[t]);
    chunk += static_cast<int>((numel[t] + kChunk - 1) / kChunk);
  }
}

int check_list(const void* const* in, const int64_t* numel, const int32_t* dtype, int32_t n, const char* what) {
  int64_t chunks = 0;
  for (int t = 0; t < n; ++t) {
    if (numel[t] < 0 || numel[t] > (static_cast<int64_t>(1) << 42))
      return fail(BPC_ERR_ARG, std::string(what) + ": element count outside [0, 2^42]");
    const int size = size_of(dtype[t]);
    if (!size) return fail(BPC_ERR_ARG, std::string(what) + ": dtype must be f32, bf16 or f16");
    if (numel[t] && !in[t]) return fail(BPC_ERR_ARG, std::string(what) + ": null tensor");
    if (reinterpret_cast<uintptr_t>(in[t]) % size) return fail(BPC_ERR_ARG, std::string(what) + ": tensor not aligned to its type");
    chunks += (numel[t] + kChunk - 1) / kChunk;
    if (chunks > 0x3fffffff) return fail(BPC_ERR_ARG, std::string(what) + ": too many elements");
  }
  return 0;
}

// No output may share memory with another tensor of the list, in or out (its own input exactly in place excepted):
// the blocks run in no order.
int check_overlap(const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
                  const int32_t* out_dtype, int32_t n) {
  struct Range {
    uintptr_t at, end;
    bool written;
  };
  std::vector<Range> r;
  r.reserve(2 * static_cast<size_t>(n));
  bool sorted = true;
  auto add = [&](const void* p, int64_t bytes, bool written) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (!r.empty() && r.back().at > at) sorted = false;
    r.push_back({at, at + static_cast<uintptr_t>(bytes), written});
  };
  for (int t = 0; t < n; ++t) {
    if (numel[t] == 0) continue;
    const bool in_place = in[t] == out[t] && in_dtype[t] == out_dtype[t];
    if (!in_place) add(in[t], numel[t] * size_of(in_dtype[t]), false);
    add(out[t], numel[t] * size_of(out_dtype[t]), true);
  }
  if (!sorted) std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.at < b.at; });
  uintptr_t read_end = 0, written_end = 0;
  for (const Range& x : r) {
    if (x.at < written_end || (x.written && x.at < read_end))
      return fail(BPC_ERR_ARG, "clip_grads: an output overlaps another tensor of the list");
    uintptr_t& end = x.written ? written_end : read_end;
    end = std::max(end, x.end);
  }
  return 0;
}

template <int N>
int launch_partial(const Part& p, const void* const* in, const int64_t* numel, const int32_t* dtype, double* partial,
                   cudaStream_t s) {
  List<N> list;
  fill(&list, p, in, nullptr, numel, dtype, nullptr);
  norm_partial_kernel<N><<<p.blocks, kThreads, 0, s>>>(list, p.per_block, partial);
  return launched("norm_partial_kernel");
}

template <int N>
int launch_scale(const Part& p, const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
                 const int32_t* out_dtype, const double* partial, int partials, double max_norm, float* norm,
                 cudaStream_t s) {
  List<N> list;
  fill(&list, p, in, out, numel, in_dtype, out_dtype);
  clip_scale_kernel<N><<<p.blocks, kThreads, 0, s>>>(list, p.per_block, partial, partials, max_norm, norm);
  return launched("clip_scale_kernel");
}

// The partial sums of every launch; *partials counts them
int run_partials(const std::vector<Part>& parts, const void* const* in, const int64_t* numel, const int32_t* dtype,
                 double* partial, int* partials, cudaStream_t s) {
  *partials = 0;
  for (const Part& p : parts) {
    if (!p.blocks) continue;
    const int n = p.t1 - p.t0;
    double* at = partial + *partials;
    const int e = n <= 32 ? launch_partial<32>(p, in, numel, dtype, at, s)
                          : n <= 200 ? launch_partial<200>(p, in, numel, dtype, at, s)
                                     : launch_partial<kListMax>(p, in, numel, dtype, at, s);
    if (e) return e;
    *partials += p.blocks;
  }
  return 0;
}

int finish(const double* partial, int partials, float* norm, cudaStream_t s) {
  norm_finish_kernel<<<1, kThreads, 0, s>>>(partial, partials, norm);
  return launched("norm_finish_kernel");
}

int check_common(const void* const* tensors, const int64_t* numel, const int32_t* dtype, int32_t n, float* norm,
                 void* workspace, size_t workspace_bytes, const char* what) {
  if (n < 0 || n > (1 << 20)) return fail(BPC_ERR_ARG, std::string(what) + ": 0 <= n <= 2^20 tensors");
  if (!norm || !workspace || (n && (!tensors || !numel || !dtype))) return fail(BPC_ERR_ARG, std::string(what) + ": null buffer");
  if ((reinterpret_cast<uintptr_t>(norm) & 3) || (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(BPC_ERR_ARG, std::string(what) + ": norm must be 4-byte and the workspace 8-byte aligned");
  if (workspace_bytes < bpc_grad_norm_workspace_size(n)) return fail(BPC_ERR_SPACE, std::string(what) + ": workspace too small");
  return check_list(tensors, numel, dtype, n, what);
}

}  // namespace

}  // namespace bpc

using namespace bpc;

extern "C" size_t bpc_grad_norm_workspace_size(int32_t n) {
  if (n < 0 || n > (1 << 20)) return 0;
  return sizeof(double) * static_cast<size_t>(max_blocks()) * std::max(1, launches_of(n));
}

extern "C" int bpc_grad_norm(const void* const* tensors, const int64_t* numel, const int32_t* dtype, int32_t n,
                             float* norm, void* workspace, size_t workspace_bytes, bpc_stream_t stream) {
  if (int e = check_common(tensors, numel, dtype, n, norm, workspace, workspace_bytes, "grad_norm")) return e;
  try {
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(workspace);
    int partials = 0;
    if (int e = run_partials(parts_of(numel, n), tensors, numel, dtype, partial, &partials, s)) return e;
    return finish(partial, partials, norm, s);
  } catch (const std::exception& e) {      // a host array that cannot be allocated
    return fail(BPC_ERR_ARG, e.what());
  }
}

extern "C" int bpc_clip_grads(const void* const* tensors, void* const* out, const int64_t* numel, const int32_t* dtype,
                              const int32_t* out_dtype, int32_t n, double max_norm, float* norm, void* workspace,
                              size_t workspace_bytes, bpc_stream_t stream) {
  if (!(max_norm >= 0)) return fail(BPC_ERR_ARG, "clip_grads: max_norm must not be negative or NaN");
  if (int e = check_common(tensors, numel, dtype, n, norm, workspace, workspace_bytes, "clip_grads")) return e;
  if (n && (!out || !out_dtype)) return fail(BPC_ERR_ARG, "clip_grads: null buffer");
  if (int e = check_list(const_cast<const void* const*>(out), numel, out_dtype, n, "clip_grads output")) return e;
  try {
    if (int e = check_overlap(tensors, out, numel, dtype, out_dtype, n)) return e;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(workspace);
    int partials = 0;
    const std::vector<Part> parts = parts_of(numel, n);
    if (int e = run_partials(parts, tensors, numel, dtype, partial, &partials, s)) return e;
    if (!partials) return finish(partial, 0, norm, s);
    for (const Part& p : parts) {
      if (!p.blocks) continue;
      const int k = p.t1 - p.t0;
      const int e = k <= 32 ? launch_scale<32>(p, tensors, out, numel, dtype, out_dtype, partial, partials, max_norm, norm, s)
                    : k <= 200 ? launch_scale<200>(p, tensors, out, numel, dtype, out_dtype, partial, partials, max_norm, norm, s)
                               : launch_scale<kListMax>(p, tensors, out, numel, dtype, out_dtype, partial, partials, max_norm, norm, s);
      if (e) return e;
    }
    return 0;
  } catch (const std::exception& e) {
    return fail(BPC_ERR_ARG, e.what());
  }
}
