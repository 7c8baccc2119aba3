// What the forward and the backward kernels of the group normalisation share: types, the activation, the cut of the
// features into pieces of work, reductions.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "bpc.h"
#include "bpc_common.cuh"
#include "bpc_internal.h"

namespace bpc {
namespace gn {

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
  __device__ __forceinline__ float get(int e) const { return load_f32(&v[e]); }
  __device__ __forceinline__ void set(int e, float f) { store_f32(&v[e], f); }
};

// s(u) = 1 / (1 + e^-u); relative errors of a few 2^-24 and |u| 2^-23, whatever u is
__device__ __forceinline__ float logistic(float u) { return __fdividef(1.0f, 1.0f + __expf(-u)); }

// act(z) = z s(u), act'(z) = s + z s (1 - s) u'
constexpr float kGelu = 1.5957691216057308f;      // 2 sqrt(2 / pi)
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == BPC_ACT_NONE) return z;
  else if constexpr (ACT == BPC_ACT_SILU) return z * logistic(z);
  else return z * logistic(kGelu * z * fmaf(0.044715f * z, z, 1.0f));
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if constexpr (ACT == BPC_ACT_NONE) {
    return 1.0f;
  } else if constexpr (ACT == BPC_ACT_SILU) {
    const float s = logistic(z);
    return fmaf(z * s, 1.0f - s, s);
  } else {
    const float s = logistic(kGelu * z * fmaf(0.044715f * z, z, 1.0f));
    return fmaf(z * s * (1.0f - s), kGelu * fmaf(3.0f * 0.044715f * z, z, 1.0f), s);
  }
}

struct Shape {
  int64_t B, N;
  int C, G;
  int64_t x_sample, x_row;        // strides in elements
  int64_t g_sample, g_row;        // of gy
};

// How the features are cut.
//   units  small samples: `lanes` neighbouring lanes take a sample's group, `slots` vectors each, `rows` samples a block
//   tiles  a block takes some rows (a chunk) of a slab of whole groups of one sample in its registers, a thread always the
//          same channels: V threads across, `lanes` down, kRows rows a thread at most.  The chunks of a sample are a cluster
//          that exchanges its sums (up to kCluster blocks), or two kernels with the sums in memory between them.
//   wide   groups too wide for a row of threads: a block per sample and group in loops
enum Kind { kUnits, kTiles, kWide };
constexpr int kCluster = 8;
struct Plan {
  Kind kind;
  int vec;                        // elements per access
  int lanes, slots, rows;         // units
  int slab, slabs, V;             // tiles: channels of a slab, slabs, threads across one
  int chunks, chunk_rows;
  bool fused;
  int threads;
};

constexpr int kMaxThreads = 512;

// rows a thread holds; whole-width accesses need everything on 16-byte boundaries (`aligned`)
inline Plan make_plan(const Shape& s, int size, int k_rows, int sms, bool aligned) {
  Plan p = {};
  const int cg = s.C / s.G, full = 16 / size;
  p.vec = aligned && cg % full == 0 ? full : 1;
  const int across = cg / p.vec;
  // small samples, of which a block per sample and slab would have little: 32-byte pieces of rows at least, or whole rows
  const int64_t vectors = s.N * across;
  if (vectors <= 128 && (s.N == 1 || cg * size >= 32)) {
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes < vectors) p.lanes *= 2;
    p.slots = vectors <= p.lanes ? 1 : 4;
    if (static_cast<int64_t>(p.lanes) * s.G <= kMaxThreads) {
      p.kind = kUnits;
      p.rows = std::max(1, 256 / (p.lanes * s.G));
      p.threads = (p.lanes * s.G * p.rows + 31) / 32 * 32;
      return p;
    }
  }
  if (across > kMaxThreads) {
    p.kind = kWide;
    p.threads = 256;
    return p;
  }
  p.kind = kTiles;
  // slabs of 64-byte rows or one group, whichever is wider
  const int groups = std::min(s.G, std::max(1, std::min((64 / size + cg - 1) / cg, kMaxThreads / across)));
  p.slab = groups * cg;
  p.slabs = (s.G + groups - 1) / groups;
  p.V = p.slab / p.vec;
  int lanes = std::max(1, 256 / p.V);
  if (s.N > static_cast<int64_t>(lanes) * k_rows) lanes = std::max(1, kMaxThreads / p.V);
  // few blocks: more chunks, down to a row per thread
  const int64_t blocks = s.B * p.slabs;
  int64_t chunks = (s.N + static_cast<int64_t>(lanes) * k_rows - 1) / (static_cast<int64_t>(lanes) * k_rows);
  if (chunks <= kCluster) {
    while (chunks < kCluster && blocks * chunks * 2 <= sms && s.N >= lanes * chunks * 2) chunks *= 2;
    chunks = std::min<int64_t>(chunks, kCluster);
  }
  p.fused = chunks <= kCluster;
  p.chunk_rows = static_cast<int>((s.N + chunks - 1) / chunks);
  p.chunks = static_cast<int>((s.N + p.chunk_rows - 1) / p.chunk_rows);
  p.threads = (std::min(lanes, p.chunk_rows) * p.V + 31) / 32 * 32;
  return p;
}

// Sums over the threads of each group of a slab: thread (row r, vector v) has v, groups of `across` vectors; the sums of
// group j come out in out[j].  part: a float per thread.
__device__ __forceinline__ void group_sums(float value, int V, int rows, int across, int groups, float* part, float* out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int entries = rows;
  if (V <= 32 && (V & (V - 1)) == 0) {
    for (int d = 16; d >= V; d >>= 1) value += __shfl_xor_sync(0xffffffffu, value, d);
    if (lane < V) part[warp * V + lane] = value;
    entries = warps;
  } else if (threadIdx.x < rows * V) {
    part[threadIdx.x] = value;
  }
  __syncthreads();
  for (int j = warp; j < groups; j += warps) {
    float sum = 0.0f;
    for (int i = lane; i < entries * across; i += 32) sum += part[i / across * V + j * across + i % across];
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) out[j] = sum;
  }
  __syncthreads();
}

inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

// One launch, as clusters of `cluster` blocks
inline int launch(const void* fn, unsigned grid, int threads, int cluster, cudaStream_t s, void** args, const char* what) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(grid);
  lc.blockDim = dim3(threads);
  lc.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelExC(&lc, fn, args);
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

inline int size_of(int32_t dtype) { return dtype == BPC_DTYPE_F32 ? 4 : dtype == BPC_DTYPE_BF16 || dtype == BPC_DTYPE_F16 ? 2 : 0; }

template <typename T>
struct Type {
  typedef T type;
};
// The pairs of types that occur: equal ones, and fp32 features with a bf16 or fp16 result.
template <typename F>
int with_types(int32_t x, int32_t y, F f) {
  if (x == BPC_DTYPE_F32) {
    if (y == BPC_DTYPE_F32) return f(Type<float>(), Type<float>());
    if (y == BPC_DTYPE_BF16) return f(Type<float>(), Type<__nv_bfloat16>());
    return f(Type<float>(), Type<__half>());
  }
  if (x == BPC_DTYPE_BF16) return f(Type<__nv_bfloat16>(), Type<__nv_bfloat16>());
  return f(Type<__half>(), Type<__half>());
}
template <typename F>
int with_act(int32_t act, F f) {
  if (act == BPC_ACT_NONE) return f(std::integral_constant<int, BPC_ACT_NONE>());
  if (act == BPC_ACT_SILU) return f(std::integral_constant<int, BPC_ACT_SILU>());
  return f(std::integral_constant<int, BPC_ACT_GELU>());
}

inline bool aligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// Strides of a (B, N, C) tensor with contiguous channels: not negative (0 broadcasts)
inline bool stride_ok(int64_t s) { return s >= 0 && s <= (static_cast<int64_t>(1) << 40); }

inline int check_shape(const Shape& s, int32_t act, int32_t x_dtype, int32_t y_dtype, const char* what) {
  auto bad = [&](const char* m) { return fail(BPC_ERR_ARG, std::string(what) + ": " + m); };
  if (s.B < 0 || s.N < 0 || s.B > (static_cast<int64_t>(1) << 40) || s.N > (static_cast<int64_t>(1) << 30) ||
      (s.N && s.B > (static_cast<int64_t>(1) << 40) / s.N))
    return bad("samples x rows outside [0, 2^40], or rows beyond 2^30");
  if (s.C < 1 || s.C > (1 << 20)) return bad("1 <= channels <= 2^20");
  if (s.G < 1 || s.C % s.G) return bad("the channels must divide into the groups");
  if (act < BPC_ACT_NONE || act > BPC_ACT_GELU) return bad("unknown activation");
  if (!size_of(x_dtype) || !size_of(y_dtype) || (x_dtype != y_dtype && x_dtype != BPC_DTYPE_F32))
    return bad("dtype must be f32, bf16 or f16, the result's the same or narrower than f32's");
  if (!stride_ok(s.x_sample) || !stride_ok(s.x_row) || !stride_ok(s.g_sample) || !stride_ok(s.g_row))
    return bad("strides outside [0, 2^40]");
  return 0;
}

// Rows of a thread's registers: 16 bytes of x each.  The backward pass keeps gz in fp32 beside x: half as many of 16-bit
// features.
constexpr int kForwardRows = 8;
inline int backward_rows(int size) { return size == 4 ? 8 : 4; }

}  // namespace gn
}  // namespace bpc
