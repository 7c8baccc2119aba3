// Linear attention with a decay for each head: a state that forgets at a fixed rate, over whole sequences (forward and
// backward) and one position at a time.
//
//   S_t = a S_(t-1) + k_t v_t^T,   o_t = scale q_t S_t   (a = exp(log_decay_h) per head, S (dk, dv), q, k, v rows)
//
// Forward and every gradient are one scan over rows a_t, b_t, c_t and a state X:
//   S = X + in b_t c_t^T;   out_t = out_scale a_t S;   X = a S
//   forward  a, b, c = q, k, v     X = a S_0             out_scale = scale      the last S is the new state
//   dq       a, b, c = go, v, k    X = a S_0^T           out_scale = scale
//   dk       a, b, c = v, go, q    X = gS^T, in = scale  backwards in time      (gS: the gradient of the new state)
//   dv       a, b, c = k, q, go    X = gS, in = scale    backwards in time      a times the last S is dS_0
#include <cmath>
#include <string>

#include "bpc.h"
#include "bpc_common.cuh"
#include "bpc_internal.h"

namespace bpc {

namespace {

constexpr int kThreads = 128;
constexpr int kMaxDim = 128;

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// (B, T, H, D) rows with contiguous D; strides in elements
struct Rows {
  const void* at;
  int64_t b, t, h;
};

struct Scan {
  Rows a, b, c;
  void* out;                    // contiguous (B, T, H, dc)
  const float* log_decay;
  const float* first;           // X before its decay: (B, H, da, dc), or (B, H, dc, da) where first_t
  float* last;                  // (B, H, da, dc), or null
  const void* lengths;
  int length_bytes;
  int64_t B, T;
  int H, da, dc;
  float in_scale, out_scale;
  bool reverse, first_t;
};

__device__ __forceinline__ int64_t length_of(const void* lengths, int bytes, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t n = bytes == 8 ? static_cast<const int64_t*>(lengths)[b] : static_cast<const int32_t*>(lengths)[b];
  return n < 0 ? 0 : n > T ? T : n;
}

// One block per sequence and head, a thread per column of the state, which stays in shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) scan_kernel(const Scan p) {
  extern __shared__ float S[];                          // (da, kThreads)
  __shared__ float ra[kMaxDim], rb[kMaxDim];
  const int64_t at = blockIdx.x, b = at / p.H;
  const int h = static_cast<int>(at % p.H), j = threadIdx.x;
  const int64_t n = length_of(p.lengths, p.length_bytes, b, p.T);
  const float a = expf(p.log_decay[h]);
  T* out = static_cast<T*>(p.out) + (b * p.T * p.H + h) * p.dc;
  const int64_t row = static_cast<int64_t>(p.H) * p.dc;
  const float* first = p.first ? p.first + at * p.da * p.dc : nullptr;
  const float lead = p.reverse || n == 0 ? 1.0f : a;
  for (int i = 0; i < p.da; ++i)
    S[i * kThreads + j] = first && j < p.dc ? lead * first[p.first_t ? j * p.da + i : i * p.dc + j] : 0.0f;
  for (int64_t k = 0; k < n; ++k) {
    const int64_t t = p.reverse ? n - 1 - k : k;
    __syncthreads();
    if (j < p.da) {
      ra[j] = load_f32(static_cast<const T*>(p.a.at) + b * p.a.b + t * p.a.t + h * p.a.h + j);
      rb[j] = load_f32(static_cast<const T*>(p.b.at) + b * p.b.b + t * p.b.t + h * p.b.h + j);
    }
    __syncthreads();
    if (j < p.dc) {
      const float c = p.in_scale * load_f32(static_cast<const T*>(p.c.at) + b * p.c.b + t * p.c.t + h * p.c.h + j);
      const float keep = k ? a : 1.0f;
      float o = 0.0f;
      for (int i = 0; i < p.da; ++i) {
        const float s = fmaf(rb[i], c, keep * S[i * kThreads + j]);
        S[i * kThreads + j] = s;
        o = fmaf(ra[i], s, o);
      }
      store_f32(out + t * row + j, p.out_scale * o);
    }
  }
  if (j < p.dc) {
    for (int64_t t = n; t < p.T; ++t) store_f32(out + t * row + j, 0.0f);
    if (p.last)
      for (int i = 0; i < p.da; ++i)
        p.last[(at * p.da + i) * p.dc + j] = (p.reverse && n ? a : 1.0f) * S[i * kThreads + j];
  }
}

// One block per sequence and head: the state updated and read once.
template <typename T>
__global__ void __launch_bounds__(kThreads) step_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                        const T* __restrict__ v, T* __restrict__ o,
                                                        const float* __restrict__ log_decay, const float* state,
                                                        float* new_state, int H, int dk, int dv, int64_t qb, int64_t qh,
                                                        int64_t kb, int64_t kh, int64_t vb, int64_t vh, float scale) {
  const int64_t at = blockIdx.x, b = at / H;
  const int h = static_cast<int>(at % H), j = threadIdx.x;
  if (j >= dv) return;
  const float a = expf(log_decay[h]), c = load_f32(v + b * vb + h * vh + j);
  float sum = 0.0f;
  for (int i = 0; i < dk; ++i) {
    const int64_t e = (at * dk + i) * dv + j;
    const float s = fmaf(load_f32(k + b * kb + h * kh + i), c, a * state[e]);
    new_state[e] = s;
    sum = fmaf(load_f32(q + b * qb + h * qh + i), s, sum);
  }
  store_f32(o + at * dv + j, scale * sum);
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

int size_of(int32_t dtype) { return dtype == BPC_DTYPE_F32 ? 4 : dtype == BPC_DTYPE_BF16 ? 2 : 0; }

bool aligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

int run_scan(const Scan& p, int32_t dtype, cudaStream_t s) {
  const int smem = p.da * kThreads * static_cast<int>(sizeof(float));
  const void* fn = dtype == BPC_DTYPE_F32 ? reinterpret_cast<const void*>(&scan_kernel<float>)
                                          : reinterpret_cast<const void*>(&scan_kernel<__nv_bfloat16>);
  if (int e = allow_smem(fn, smem)) return e;
  const unsigned grid = static_cast<unsigned>(p.B * p.H);
  if (dtype == BPC_DTYPE_F32) scan_kernel<float><<<grid, kThreads, smem, s>>>(p);
  else scan_kernel<__nv_bfloat16><<<grid, kThreads, smem, s>>>(p);
  return launched("linear_attention");
}

int check_common(const std::string& what, int64_t B, int64_t T, int32_t H, int32_t dk, int32_t dv, const void* lengths,
                 int32_t length_bytes, const int64_t* strides, int n_strides, float scale, int32_t dtype,
                 const float* log_decay) {
  auto bad = [&](const char* m) { return fail(BPC_ERR_ARG, what + ": " + m); };
  if (B < 0 || T < 0 || H < 0 || T > (static_cast<int64_t>(1) << 31)) return bad("batch, length and heads must not be negative, length <= 2^31");
  if (H && B > 0x7fffffff / H) return bad("batch x heads must be below 2^31");
  if (dk < 1 || dk > kMaxDim || dv < 1 || dv > kMaxDim) return bad("head sizes must be 1 to 128");
  if (!size_of(dtype)) return bad("dtype must be f32 or bf16");
  if (!std::isfinite(scale)) return bad("scale must be finite");
  if (lengths && ((length_bytes != 4 && length_bytes != 8) || !aligned(lengths, length_bytes)))
    return bad("lengths must be int32 or int64");
  if (!strides) return bad("null strides");
  for (int i = 0; i < n_strides; ++i)
    if (strides[i] < 0 || strides[i] > (static_cast<int64_t>(1) << 40)) return bad("strides outside [0, 2^40]");
  if (B && H && (!log_decay || !aligned(log_decay, 4))) return bad("null or unaligned log_decay");
  return 0;
}

Rows rows_of(const void* p, const int64_t* s) { return {p, s[0], s[1], s[2]}; }

}  // namespace

}  // namespace bpc

using namespace bpc;

extern "C" size_t bpc_linear_attention_workspace_size(int64_t B, int64_t T, int32_t H, int32_t dk, int32_t dv,
                                                      int32_t dtype, int32_t backward) {
  if (B < 1 || T < 0 || H < 1 || dk < 1 || dk > kMaxDim || dv < 1 || dv > kMaxDim || !size_of(dtype)) return 0;
  return 16;
}

extern "C" int bpc_linear_attention_fwd(const void* q, const void* k, const void* v, void* o, const float* log_decay,
                                        const float* state, float* new_state, const void* lengths, int32_t length_bytes,
                                        int64_t B, int64_t T, int32_t H, int32_t dk, int32_t dv, const int64_t* strides,
                                        float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                                        bpc_stream_t stream) {
  const char* what = "linear_attention";
  if (int e = check_common(what, B, T, H, dk, dv, lengths, length_bytes, strides, 9, scale, dtype, log_decay)) return e;
  if (B == 0 || H == 0 || (T == 0 && !new_state)) return 0;
  const int size = size_of(dtype);
  if ((T && (!q || !k || !v || !o)) || !workspace) return fail(BPC_ERR_ARG, "linear_attention: null buffer");
  if (!aligned(q, size) || !aligned(k, size) || !aligned(v, size) || !aligned(o, size) || !aligned(state, 16) ||
      !aligned(new_state, 16) || !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "linear_attention: buffer not aligned to its type (states and workspace: 16 bytes)");
  if (workspace_bytes < bpc_linear_attention_workspace_size(B, T, H, dk, dv, dtype, 0))
    return fail(BPC_ERR_SPACE, "linear_attention: workspace too small");
  const Scan p{rows_of(q, strides), rows_of(k, strides + 3), rows_of(v, strides + 6), o, log_decay, state, new_state, lengths,
               length_bytes, B, T, H, dk, dv, 1.0f, scale, false, false};
  return run_scan(p, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int bpc_linear_attention_bwd(const void* q, const void* k, const void* v, const void* go, const float* log_decay,
                                        const float* state, const float* grad_state, const void* lengths,
                                        int32_t length_bytes, void* dq, void* dk_out, void* dv_out, float* dstate, int64_t B,
                                        int64_t T, int32_t H, int32_t dk, int32_t dv, const int64_t* strides, float scale,
                                        int32_t dtype, void* workspace, size_t workspace_bytes, bpc_stream_t stream) {
  const char* what = "linear_attention backward";
  if (int e = check_common(what, B, T, H, dk, dv, lengths, length_bytes, strides, 12, scale, dtype, log_decay)) return e;
  if (B == 0 || H == 0 || (T == 0 && !dstate)) return 0;
  const int size = size_of(dtype);
  if ((T && (!q || !k || !v || !go || !dq || !dk_out || !dv_out)) || !workspace)
    return fail(BPC_ERR_ARG, "linear_attention backward: null buffer");
  for (const void* b : {q, k, v, go, static_cast<const void*>(dq), static_cast<const void*>(dk_out), static_cast<const void*>(dv_out)})
    if (!aligned(b, size)) return fail(BPC_ERR_ARG, "linear_attention backward: buffer not aligned to its type");
  if (!aligned(state, 16) || !aligned(grad_state, 16) || !aligned(dstate, 16) || !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "linear_attention backward: buffer not aligned to its type (states and workspace: 16 bytes)");
  if (workspace_bytes < bpc_linear_attention_workspace_size(B, T, H, dk, dv, dtype, 1))
    return fail(BPC_ERR_SPACE, "linear_attention backward: workspace too small");
  const Rows rq = rows_of(q, strides), rk = rows_of(k, strides + 3), rv = rows_of(v, strides + 6), rg = rows_of(go, strides + 9);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (T) {
    const Scan pq{rg, rv, rk, dq, log_decay, state, nullptr, lengths, length_bytes, B, T, H, dv, dk, 1.0f, scale, false, true};
    if (int e = run_scan(pq, dtype, s)) return e;
    const Scan pk{rv, rg, rq, dk_out, log_decay, grad_state, nullptr, lengths, length_bytes, B, T, H, dv, dk, scale, 1.0f, true, true};
    if (int e = run_scan(pk, dtype, s)) return e;
  }
  const Scan pv{rk, rq, rg, dv_out, log_decay, grad_state, dstate, lengths, length_bytes, B, T, H, dk, dv, scale, 1.0f, true, false};
  return run_scan(pv, dtype, s);
}

extern "C" int bpc_linear_attention_step(const void* q, const void* k, const void* v, void* o, const float* log_decay,
                                         const float* state, float* new_state, int64_t B, int32_t H, int32_t dk, int32_t dv,
                                         const int64_t* strides, float scale, int32_t dtype, bpc_stream_t stream) {
  const char* what = "linear_attention_step";
  if (int e = check_common(what, B, 1, H, dk, dv, nullptr, 0, strides, 6, scale, dtype, log_decay)) return e;
  if (B == 0 || H == 0) return 0;
  const int size = size_of(dtype);
  if (!q || !k || !v || !o || !state || !new_state) return fail(BPC_ERR_ARG, "linear_attention_step: null buffer");
  if (!aligned(q, size) || !aligned(k, size) || !aligned(v, size) || !aligned(o, size) || !aligned(state, 4) || !aligned(new_state, 4))
    return fail(BPC_ERR_ARG, "linear_attention_step: buffer not aligned to its type");
  const uintptr_t at = reinterpret_cast<uintptr_t>(state), to = reinterpret_cast<uintptr_t>(new_state);
  const uintptr_t bytes = sizeof(float) * static_cast<uintptr_t>(B) * H * dk * dv;
  if (at != to && at < to + bytes && to < at + bytes)
    return fail(BPC_ERR_ARG, "linear_attention_step: new_state overlaps state (give the same buffer to update it in place)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(B * H);
  if (dtype == BPC_DTYPE_F32)
    step_kernel<float><<<grid, kThreads, 0, s>>>(static_cast<const float*>(q), static_cast<const float*>(k),
                                                 static_cast<const float*>(v), static_cast<float*>(o), log_decay, state, new_state,
                                                 H, dk, dv, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5],
                                                 scale);
  else
    step_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(
        static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v),
        static_cast<__nv_bfloat16*>(o), log_decay, state, new_state, H, dk, dv, strides[0], strides[1], strides[2], strides[3],
        strides[4], strides[5], scale);
  return launched(what);
}
