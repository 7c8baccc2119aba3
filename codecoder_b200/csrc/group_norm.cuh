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
#include "group_norm_plan.h"

namespace bpc {
namespace gn {

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }

// VEC elements of an access, as 32-bit words.  Arithmetic is on pairs of them in fp32 (f2_* of bpc_common.cuh: half the
// instructions); a single element has a pair with a zero beside it.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  static constexpr int kPairs = VEC / 2;
  static constexpr bool kF32 = sizeof(T) == 4;
  uint32_t w[VEC * sizeof(T) / 4];
  __device__ __forceinline__ uint64_t pair(int k) const {
    if constexpr (kF32) {
      return f2_pack(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return bf2_to_f2(w[k]);
    } else {
      const float2 f = __half22float2(__halves2half2(__ushort_as_half(w[k] & 0xffff), __ushort_as_half(w[k] >> 16)));
      return f2_pack(f.x, f.y);
    }
  }
  __device__ __forceinline__ void set(int k, uint64_t x) {
    if constexpr (kF32) {
      w[2 * k] = __float_as_uint(f2_lo(x)), w[2 * k + 1] = __float_as_uint(f2_hi(x));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      w[k] = f2_to_bf2(x);
    } else {
      const __half2 h = __floats2half2_rn(f2_lo(x), f2_hi(x));
      w[k] = static_cast<uint32_t>(__half_as_ushort(__low2half(h))) | static_cast<uint32_t>(__half_as_ushort(__high2half(h))) << 16;
    }
  }
};
template <typename T>
struct alignas(sizeof(T)) Pack<T, 1> {
  static constexpr int kPairs = 1;
  T v;
  __device__ __forceinline__ uint64_t pair(int) const { return f2_pack(load_f32(&v), 0.0f); }
  __device__ __forceinline__ void set(int, uint64_t x) { store_f32(&v, f2_lo(x)); }
};
template <int VEC>
__device__ __forceinline__ float both(uint64_t x) {
  return VEC == 1 ? f2_lo(x) : f2_lo(x) + f2_hi(x);
}
__device__ __forceinline__ uint64_t f2_of(float x) { return f2_pack(x, x); }

// per-channel parameters of a vector from channel c on, `other` where there are none
template <int VEC>
__device__ __forceinline__ void channels(const float* p, int c, bool there, float other, uint64_t (&out)[(VEC + 1) / 2]) {
#pragma unroll
  for (int k = 0; k < (VEC + 1) / 2; ++k) {
    const float lo = there && p ? __ldg(p + c + 2 * k) : other;
    out[k] = f2_pack(lo, VEC == 1 ? 0.0f : there && p ? __ldg(p + c + (VEC == 1 ? 0 : 2 * k + 1)) : other);
  }
}

// s(u) = 1 / (1 + e^-u): off by a few 2^-24 and |u| 2^-23 of itself from u = -87.3 up.  Below, where s is smaller than fp32's normal
// numbers (2^-126), it is zero: z s(z) is off by at most 88 2^-126 there, absolutely
__device__ __forceinline__ uint64_t logistic(uint64_t u) {
  const uint64_t t = f2_mul(u, f2_of(-1.4426950408889634f));
  float e0, e1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(f2_lo(t)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(f2_hi(t)));
  const uint64_t d = f2_add(f2_pack(e0, e1), f2_of(1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(f2_lo(d)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(f2_hi(d)));
  return f2_pack(e0, e1);
}

// act(z) = z s(u(z)) and act'(z) = s (1 + z u' (1 - s)); z u' of the GELU is a number of fp32 for |z| up to 10^13, and its slope NaN
// beyond
constexpr float kGelu = 1.5957691216057308f;      // 2 sqrt(2 / pi)
constexpr float kGelu3 = 0.044715f * kGelu;
template <int ACT>
__device__ __forceinline__ uint64_t activate(uint64_t z) {
  if constexpr (ACT == BPC_ACT_NONE) return z;
  else if constexpr (ACT == BPC_ACT_SILU) return f2_mul(z, logistic(z));
  else return f2_mul(z, logistic(f2_mul(z, f2_fma(f2_mul(z, z), f2_of(kGelu3), f2_of(kGelu)))));
}
template <int ACT>
__device__ __forceinline__ uint64_t slope(uint64_t z) {
  if constexpr (ACT == BPC_ACT_NONE) return f2_of(1.0f);
  uint64_t s, zu = z;
  if constexpr (ACT == BPC_ACT_SILU) {
    s = logistic(z);
  } else {
    const uint64_t zz = f2_mul(z, z);
    s = logistic(f2_mul(z, f2_fma(zz, f2_of(kGelu3), f2_of(kGelu))));
    zu = f2_mul(z, f2_fma(zz, f2_of(3.0f * kGelu3), f2_of(kGelu)));
  }
  return f2_mul(s, f2_fma(zu, f2_fma(s, f2_of(-1.0f), f2_of(1.0f)), f2_of(1.0f)));
}
// the wide kernels' single values
template <int ACT>
__device__ __forceinline__ float activate1(float z) {
  return f2_lo(activate<ACT>(f2_pack(z, 0.0f)));
}
template <int ACT>
__device__ __forceinline__ float slope1(float z) {
  return f2_lo(slope<ACT>(f2_pack(z, 0.0f)));
}

// sum / n with per = 1 / n rounded: the quotient of a product and its remainder, exact where the quotient is a number of fp32
__device__ __forceinline__ float over(float sum, float n, float per) {
  const float q = sum * per;
  return fmaf(fmaf(-q, n, sum), per, q);
}

// the sum over `lanes` neighbouring lanes, in each of them; the steps written out: a loop of them costs as much again
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
#pragma unroll
  for (int m = 1; m < 32; m *= 2)
    if (lanes > m) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// 1 / sqrt(v) to within 2^-23: the approximation and one step of Newton's, but at the ends, where that has no value
__device__ __forceinline__ float inverse_sqrt(float v) {
  const float r = rsqrtf(v), n = r * fmaf(-0.5f * v * r, r, 1.5f);
  return v > 1e-30f && v < 1e30f ? n : 1.0f / sqrtf(v);
}

// The sums of N values over the threads of the calling thread's group of a slab, in each of them: thread (row r, vector v) has
// vector v of V, groups of `across` vectors.  part: N floats per tile thread, free again after the next barrier but one.
template <int N>
__device__ __forceinline__ void group_sums(float (&value)[N], int V, int rows, int across, int v, float* part) {
  constexpr int kWarps = kTileThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = v / across;
  if (V <= 32 && (V & (V - 1)) == 0) {             // so is across: a warp's lanes of a group join by shuffles
    const int joins = ~(V - 1) | (across - 1);     // the bits of the lane that its group does not say
#pragma unroll
    for (int d = 16; d; d >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float t = __shfl_xor_sync(0xffffffffu, value[k], d);
        value[k] += d & joins ? t : 0.0f;
      }
    // [value][group][warp]
    if (lane < V && lane % across == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) part[k * kTileThreads + lane / across * kWarps + warp] = value[k];
    }
    __syncthreads();
    const int warps = blockDim.x >> 5;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float* f = part + k * kTileThreads + j * kWarps;
      float4 a = *reinterpret_cast<const float4*>(f), b = *reinterpret_cast<const float4*>(f + 4);
      if (warps < kWarps) {
        a = make_float4(a.x, warps > 1 ? a.y : 0.0f, warps > 2 ? a.z : 0.0f, warps > 3 ? a.w : 0.0f);
        b = make_float4(warps > 4 ? b.x : 0.0f, warps > 5 ? b.y : 0.0f, warps > 6 ? b.z : 0.0f, 0.0f);
      }
      value[k] = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
    }
    return;
  }
  if (threadIdx.x < rows * V) {
#pragma unroll
    for (int k = 0; k < N; ++k) part[k * kTileThreads + threadIdx.x] = value[k];
  }
  __syncthreads();
  // a warp per group; the sums go where its first thread's values were, when all of them are read
  const int down = 32 / across, along = 32 % across;
  for (int g = warp; g < V / across; g += blockDim.x >> 5) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float* f = part + k * kTileThreads + g * across;
      float sum = 0.0f;
      for (int row = lane / across, col = lane % across; row < rows;) {      // entries lane, lane + 32, ... of rows of `across`
        sum += f[row * V + col];
        row += down, col += along;
        if (col >= across) col -= across, ++row;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) f[0] = sum;                   // read by this warp alone until here
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) value[k] = part[k * kTileThreads + j * across];
}

// The mean of n values of which each of a block's 256 threads has added its own, in every thread; red: 8 numbers.  In 64 bits, as a
// wide group's thread adds N C / (256 G) values one after the other (120,000 of 30,000 rows of 1,021 channels).
__device__ __forceinline__ float block_mean(double v, int64_t n, double* red) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += red[w];
  __syncthreads();
  return static_cast<float>(s / static_cast<double>(n));
}

// f(a constant true or false): whether all of a thread's rows are there, so that most threads need not ask for each
template <typename F>
__device__ __forceinline__ void with_rows(bool all, F f) {
  if (all) f(std::true_type());
  else f(std::false_type());
}

__device__ __forceinline__ void cp_async(void* dst, const void* src, std::integral_constant<int, 16>) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async(void* dst, const void* src, std::integral_constant<int, 8>) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Vectors of the next samples on their way through shared memory, each read by the thread that fetched it: no
// barrier, and no registers (one sample ahead in those kept too little under way).  A stage holds what the block's threads
// fetch of a sample each; copies cannot take single elements of 2 bytes, which are read when used.
template <typename T, int VEC>
struct Copied {
  using P = Pack<T, VEC>;
  static constexpr int kBytes = copied_bytes(sizeof(T), VEC);
  static constexpr bool kCopies = kBytes > 0;
  __device__ static __forceinline__ void fetch(uint32_t at, const T* src) {
    if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(src) : "memory");
    else if constexpr (kBytes > 0) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(src), "n"(kBytes) : "memory");
  }
  __device__ static __forceinline__ P take(const uint8_t* smem, uint32_t at, const T* src) {
    if constexpr (kCopies) return *reinterpret_cast<const P*>(smem + at);
    else return *reinterpret_cast<const P*>(src);
  }
};

// A thread's rows of the next piece of work on their way through shared memory, K vectors of its own (no barrier): fetch
// starts the copies, take waits for them.  Single elements are read when taken.
template <typename T, int VEC, int K>
struct Ahead {
  static constexpr bool kStaged = VEC > 1;
  static constexpr int kBytes = kStaged ? K * static_cast<int>(sizeof(T)) * VEC : 0;      // per thread
  using P = Pack<T, VEC>;
  P* at;
  const T* from;
  int64_t step;
  int n;
  __device__ __forceinline__ explicit Ahead(uint8_t* smem) : at(reinterpret_cast<P*>(smem) + threadIdx.x), from(nullptr), step(0), n(0) {}
  // n of K vectors, `step` elements apart
  __device__ __forceinline__ void fetch(const T* src, int64_t step_, int n_) {
    from = src, step = step_, n = n_;
    if constexpr (kStaged) {
      with_rows(n == K, [&](auto all) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (decltype(all)::value || k < n) cp_async(at + k * kTileThreads, src, std::integral_constant<int, static_cast<int>(sizeof(P))>());
          src += step;
        }
      });
    }
  }
  __device__ __forceinline__ void take(P (&d)[K]) const {
    if constexpr (kStaged) {
#pragma unroll
      for (int k = 0; k < K; ++k) d[k] = at[k * kTileThreads];      // without meaning behind n
    } else {
      const T* src = from;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (k < n) d[k] = *reinterpret_cast<const P*>(src);
        src += step;
      }
    }
  }
};

inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

// Blocks of x, y: every slab and chunk, and the samples that a slab's blocks walk at once; `per_sm` blocks of 256 threads, and
// more where one would walk more than `walk` samples
inline dim3 tiles_grid(const Shape& s, const Plan& p, int per_sm, int sms, int64_t walk) {
  const int64_t across = static_cast<int64_t>(p.slabs) * p.chunks;
  const int64_t resident = static_cast<int64_t>(sms) * std::max(1, per_sm * 256 / p.threads);
  return dim3(static_cast<unsigned>(across), static_cast<unsigned>(std::min<int64_t>({s.B, 65535, std::max<int64_t>({1, resident / across, (s.B + walk - 1) / walk})})));
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

}  // namespace gn
}  // namespace bpc
