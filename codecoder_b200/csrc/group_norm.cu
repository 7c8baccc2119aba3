// Group normalisation with an activation over channels-last features, and its gradients.
//
//   x (B, N, C), group g = channels [g C / G, (g + 1) C / G):  mean, var over the N C / G values of a sample and group
//   xh = (x - mean) rstd, rstd = 1 / sqrt(var + eps);   z = w_c xh + b_c;   y = act(z) = z s(u(z))
//     act: none (s = 1), SiLU (u = z), GELU in its tanh form (u = 2 sqrt(2 / pi) (z + 0.044715 z^3)), s the logistic
//     function
//   backward, gz = gy act'(z), A_c = sum_n gz, B_c = sum_n gz xh over a sample, s1 = sum_c w_c A_c, s2 = sum_c w_c B_c
//   over its group:
//     dx = rstd (gz w_c - (s1 + xh s2) / (N C / G));   dw_c = sum_b B_c;   db_c = sum_b A_c
//
// The variance is the mean of the squared differences from the mean (two passes), never a difference of squares.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include <cuda_fp16.h>

#include "bpc.h"
#include "bpc_common.cuh"
#include "bpc_internal.h"

namespace bpc {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float logistic(float u) { return 1.0f / (1.0f + __expf(-u)); }

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

// the sum over the block, in every thread; red: kThreads / 32 floats
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}

struct Shape {
  int64_t B, N;
  int C, G;
  int64_t x_sample, x_row;        // strides in elements
  int64_t g_sample, g_row;        // of gy
};

// one block per sample and group
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(kThreads) forward_kernel(const T* __restrict__ x, U* __restrict__ y, float* mean_out,
                                                           float* rstd_out, const float* __restrict__ w,
                                                           const float* __restrict__ bias, Shape s, float eps) {
  __shared__ float red[kThreads / 32];
  const int cg = s.C / s.G;
  const int64_t n = s.N * cg;
  for (int64_t at = blockIdx.x; at < s.B * s.G; at += gridDim.x) {
    const int64_t b = at / s.G;
    const int c0 = static_cast<int>(at % s.G) * cg;
    const T* xs = x + b * s.x_sample + c0;
    float sum = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) sum += load_f32(xs + i / cg * s.x_row + i % cg);
    const float mean = block_sum(sum, red) / static_cast<float>(n);
    float sq = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
      const float d = load_f32(xs + i / cg * s.x_row + i % cg) - mean;
      sq = fmaf(d, d, sq);
    }
    const float rstd = 1.0f / sqrtf(block_sum(sq, red) / static_cast<float>(n) + eps);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[at] = mean;
      if (rstd_out) rstd_out[at] = rstd;
    }
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      const float z = fmaf(w ? w[c] : 1.0f, xh, bias ? bias[c] : 0.0f);
      store_f32(y + (b * s.N + r) * s.C + c, activate<ACT>(z));
    }
  }
}

template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(kThreads) backward_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                            const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                            const float* __restrict__ bias, T* __restrict__ dx, Shape s) {
  __shared__ float red[kThreads / 32];
  const int cg = s.C / s.G;
  const int64_t n = s.N * cg;
  for (int64_t at = blockIdx.x; at < s.B * s.G; at += gridDim.x) {
    const int64_t b = at / s.G;
    const int c0 = static_cast<int>(at % s.G) * cg;
    const float mean = mean_in[at], rstd = rstd_in[at];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float wc = w ? w[c] : 1.0f;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      const float a = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope<ACT>(fmaf(wc, xh, bias ? bias[c] : 0.0f)) * wc;
      s1 += a;
      s2 = fmaf(a, xh, s2);
    }
    s1 = block_sum(s1, red) / static_cast<float>(n);
    s2 = block_sum(s2, red) / static_cast<float>(n);
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float wc = w ? w[c] : 1.0f;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      const float a = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope<ACT>(fmaf(wc, xh, bias ? bias[c] : 0.0f)) * wc;
      store_f32(dx + (b * s.N + r) * s.C + c, rstd * (a - fmaf(xh, s2, s1)));
    }
  }
}

// one block per channel, 64-bit sums
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(kThreads) weight_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                          const float* __restrict__ bias, float* __restrict__ dw,
                                                          float* __restrict__ db, Shape s) {
  __shared__ double red[2][kThreads / 32];
  const int c = blockIdx.x, cg = s.C / s.G, g = c / cg;
  const float wc = w ? w[c] : 1.0f, bc = bias ? bias[c] : 0.0f;
  double a = 0.0, d = 0.0;
  for (int64_t i = threadIdx.x; i < s.B * s.N; i += kThreads) {
    const int64_t b = i / s.N, r = i % s.N;
    const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean_in[b * s.G + g]) * rstd_in[b * s.G + g];
    const float gz = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope<ACT>(fmaf(wc, xh, bc));
    a += gz;
    d += static_cast<double>(gz) * xh;
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, m);
    d += __shfl_xor_sync(0xffffffffu, d, m);
  }
  if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = a, red[1][threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kThreads / 32; ++k) a += red[0][k], d += red[1][k];
    if (db) db[c] = static_cast<float>(a);
    if (dw) dw[c] = static_cast<float>(d);
  }
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

int size_of(int32_t dtype) { return dtype == BPC_DTYPE_F32 ? 4 : dtype == BPC_DTYPE_BF16 || dtype == BPC_DTYPE_F16 ? 2 : 0; }

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

bool aligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// Strides of a (B, N, C) tensor with contiguous channels: non-negative (0 broadcasts), rows apart by C or more or broadcast
bool stride_ok(int64_t s) { return s >= 0 && s <= (static_cast<int64_t>(1) << 40); }

int check_shape(const Shape& s, int32_t act, int32_t x_dtype, int32_t y_dtype, const char* what) {
  auto bad = [&](const char* m) { return fail(BPC_ERR_ARG, std::string(what) + ": " + m); };
  if (s.B < 0 || s.N < 0 || s.B > (static_cast<int64_t>(1) << 40) || s.N > (static_cast<int64_t>(1) << 40) ||
      (s.N && s.B > (static_cast<int64_t>(1) << 40) / s.N))
    return bad("samples x rows outside [0, 2^40]");
  if (s.C < 1 || s.C > (1 << 20)) return bad("1 <= channels <= 2^20");
  if (s.G < 1 || s.C % s.G) return bad("the channels must divide into the groups");
  if (act < BPC_ACT_NONE || act > BPC_ACT_GELU) return bad("unknown activation");
  if (!size_of(x_dtype) || !size_of(y_dtype) || (x_dtype != y_dtype && x_dtype != BPC_DTYPE_F32))
    return bad("dtype must be f32, bf16 or f16, the result's the same or narrower than f32's");
  if (!stride_ok(s.x_sample) || !stride_ok(s.x_row) || !stride_ok(s.g_sample) || !stride_ok(s.g_row))
    return bad("strides outside [0, 2^40]");
  return 0;
}

}  // namespace

}  // namespace bpc

using namespace bpc;

extern "C" size_t bpc_group_norm_workspace_size(int64_t B, int64_t N, int32_t C, int32_t G, int32_t backward) {
  if (B < 1 || N < 1 || C < 1 || G < 1 || C % G) return 0;
  return 16;
}

extern "C" int bpc_group_norm_fwd(const void* x, void* y, float* mean, float* rstd, const float* weight, const float* bias,
                                  int64_t B, int64_t N, int32_t C, int32_t G, int64_t x_sample_stride,
                                  int64_t x_row_stride, float eps, int32_t activation, int32_t x_dtype, int32_t y_dtype,
                                  void* workspace, size_t workspace_bytes, bpc_stream_t stream) {
  const Shape s{B, N, C, G, x_sample_stride, x_row_stride, 0, 0};
  const char* what = "group_norm";
  if (int e = check_shape(s, activation, x_dtype, y_dtype, what)) return e;
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(BPC_ERR_ARG, "group_norm: eps must be finite and not negative");
  if (B == 0 || N == 0) return 0;
  if (!x || !y || !workspace) return fail(BPC_ERR_ARG, "group_norm: null buffer");
  if (!aligned(x, size_of(x_dtype)) || !aligned(y, size_of(y_dtype)) || !aligned(mean, 4) || !aligned(rstd, 4) ||
      !aligned(weight, 4) || !aligned(bias, 4) || !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "group_norm: buffer not aligned to its type (workspace: 16 bytes)");
  if (workspace_bytes < bpc_group_norm_workspace_size(B, N, C, G, 0)) return fail(BPC_ERR_SPACE, "group_norm: workspace too small");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int grid = static_cast<int>(std::min<int64_t>(B * G, 8 * num_sms()));
  return with_types(x_dtype, y_dtype, [&](auto xt, auto yt) {
    return with_act(activation, [&](auto act) {
      typedef typename decltype(xt)::type T;
      typedef typename decltype(yt)::type U;
      forward_kernel<T, U, decltype(act)::value><<<grid, kThreads, 0, st>>>(
          static_cast<const T*>(x), static_cast<U*>(y), mean, rstd, weight, bias, s, eps);
      return launched("group_norm");
    });
  });
}

extern "C" int bpc_group_norm_bwd(const void* gy, const void* x, const float* mean, const float* rstd, const float* weight,
                                  const float* bias, void* dx, float* dw, float* db, int64_t B, int64_t N, int32_t C,
                                  int32_t G, int64_t gy_sample_stride, int64_t gy_row_stride, int64_t x_sample_stride,
                                  int64_t x_row_stride, int32_t activation, int32_t x_dtype, int32_t y_dtype,
                                  void* workspace, size_t workspace_bytes, bpc_stream_t stream) {
  const Shape s{B, N, C, G, x_sample_stride, x_row_stride, gy_sample_stride, gy_row_stride};
  const char* what = "group_norm backward";
  if (int e = check_shape(s, activation, x_dtype, y_dtype, what)) return e;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!aligned(dw, 4) || !aligned(db, 4)) return fail(BPC_ERR_ARG, "group_norm backward: buffer not aligned to its type");
  if (B == 0 || N == 0) {
    if (dw && cudaMemsetAsync(dw, 0, sizeof(float) * C, st) != cudaSuccess) return launched(what);
    if (db && cudaMemsetAsync(db, 0, sizeof(float) * C, st) != cudaSuccess) return launched(what);
    return 0;
  }
  if (!gy || !x || !mean || !rstd || !workspace) return fail(BPC_ERR_ARG, "group_norm backward: null buffer");
  if (!aligned(x, size_of(x_dtype)) || !aligned(dx, size_of(x_dtype)) || !aligned(gy, size_of(y_dtype)) ||
      !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(weight, 4) || !aligned(bias, 4) || !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "group_norm backward: buffer not aligned to its type (workspace: 16 bytes)");
  if (workspace_bytes < bpc_group_norm_workspace_size(B, N, C, G, 1))
    return fail(BPC_ERR_SPACE, "group_norm backward: workspace too small");
  const int grid = static_cast<int>(std::min<int64_t>(B * G, 8 * num_sms()));
  return with_types(x_dtype, y_dtype, [&](auto xt, auto yt) {
    return with_act(activation, [&](auto act) {
      typedef typename decltype(xt)::type T;
      typedef typename decltype(yt)::type U;
      constexpr int ACT = decltype(act)::value;
      if (dx) {
        backward_kernel<T, U, ACT><<<grid, kThreads, 0, st>>>(static_cast<const U*>(gy), static_cast<const T*>(x), mean, rstd,
                                                              weight, bias, static_cast<T*>(dx), s);
        if (int e = launched(what)) return e;
      }
      if (dw || db) {
        weight_kernel<T, U, ACT><<<C, kThreads, 0, st>>>(static_cast<const U*>(gy), static_cast<const T*>(x), mean, rstd,
                                                         weight, bias, dw, db, s);
        if (int e = launched(what)) return e;
      }
      return 0;
    });
  });
}
