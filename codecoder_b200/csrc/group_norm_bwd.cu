// Group normalisation with an activation over channels-last features: the gradients.
//
//   gz = gy act'(z), A_c = sum_n gz, B_c = sum_n gz xh over a sample, s1 = sum_c w_c A_c, s2 = sum_c w_c B_c over its
//   group (z, xh as in the forward pass):
//     dx = rstd (gz w_c - (s1 + xh s2) / (N C / G));   dw_c = sum_b B_c;   db_c = sum_b A_c
//
// One read of gy and x and one write of dx where a sample's slab fits the registers of a block or a cluster.  A thread
// always has the same channels and walks the samples, so that dw and db are sums in registers until the end: a part per
// block, joined in order in fp64 (deterministic, no atomics).
#include "group_norm.cuh"

namespace bpc {
namespace gn {
namespace {

namespace cg_ = cooperative_groups;

// The channels' sums of a block: thread (row r, vector v) has VEC channels from c on, `rows` rows of threads; into
// parts[block][2][C]
template <int VEC>
__device__ __forceinline__ void channel_sums(const float (&a)[VEC], const float (&d)[VEC], int v, int V, int r, int rows, int c, int C,
                                             bool there, float* buffer, float* parts) {
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (there) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) buffer[(r * V + v) * VEC + i] = which ? d[i] : a[i];
    }
    __syncthreads();
    if (there && r == 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        double sum = 0.0;
        for (int k = 0; k < rows; ++k) sum += buffer[(k * V + v) * VEC + i];
        parts[which * C + c + i] = static_cast<float>(sum);
      }
    }
  }
}

// Units: a sample's group per `lanes` lanes, SLOTS vectors each; a thread's slots are the same places of every sample.
template <typename T, typename U, int ACT, int VEC, int SLOTS>
__global__ void __launch_bounds__(kMaxThreads) units_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                            const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                            const float* __restrict__ bias, T* __restrict__ dx, float* parts,
                                                            const Shape s, const Plan p) {
  constexpr int kAhead = SLOTS == 1 ? 2 : 1;       // samples at a time
  extern __shared__ float buffer[];
  const int cg = s.C / s.G, across = cg / VEC, n = static_cast<int>(s.N) * cg;
  const int unit = threadIdx.x / p.lanes, l = threadIdx.x % p.lanes;
  const int g = unit % s.G, r = unit / s.G;
  const bool there = r < p.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * p.rows;
  int64_t in_x[SLOTS], in_g[SLOTS];
  int out[SLOTS];
  bool has[SLOTS];
  float wv[SLOTS][VEC], bv[SLOTS][VEC], acc_a[SLOTS][VEC], acc_b[SLOTS][VEC];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    const int e = k * p.lanes + l, row = e / across, c = g * cg + e % across * VEC;
    has[k] = there && row < s.N;
    in_x[k] = row * s.x_row + c;
    in_g[k] = row * s.g_row + c;
    out[k] = row * s.C + c;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      wv[k][i] = has[k] && w ? w[c + i] : 1.0f;
      bv[k][i] = has[k] && bias ? bias[c + i] : 0.0f;
      acc_a[k][i] = acc_b[k][i] = 0.0f;
    }
  }
  const float per = 1.0f / static_cast<float>(n);
  for (int64_t b0 = static_cast<int64_t>(blockIdx.x) * p.rows + r; b0 - r < s.B; b0 += kAhead * step) {
    Pack<T, VEC> vx[kAhead][SLOTS];
    Pack<U, VEC> vg[kAhead][SLOTS];
    float mean[kAhead], rstd[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t b = b0 + a * step;
      const bool live = there && b < s.B;
      mean[a] = live ? mean_in[b * s.G + g] : 0.0f;
      rstd[a] = live ? rstd_in[b * s.G + g] : 0.0f;
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (has[k] && live) {
          vx[a][k] = *reinterpret_cast<const Pack<T, VEC>*>(x + b * s.x_sample + in_x[k]);
          vg[a][k] = *reinterpret_cast<const Pack<U, VEC>*>(gy + b * s.g_sample + in_g[k]);
        }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t b = b0 + a * step;
      const bool live = b < s.B;
      float gz[SLOTS][VEC], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (has[k] && live) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float xh = (vx[a][k].get(i) - mean[a]) * rstd[a];
            gz[k][i] = vg[a][k].get(i) * slope<ACT>(fmaf(wv[k][i], xh, bv[k][i]));
            acc_a[k][i] += gz[k][i];
            acc_b[k][i] = fmaf(gz[k][i], xh, acc_b[k][i]);
            const float t = gz[k][i] * wv[k][i];
            s1 += t;
            s2 = fmaf(t, xh, s2);
          }
        }
      for (int d = p.lanes >> 1; d; d >>= 1) {
        s1 += __shfl_xor_sync(0xffffffffu, s1, d);
        s2 += __shfl_xor_sync(0xffffffffu, s2, d);
      }
      s1 *= per, s2 *= per;
      if (dx) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k)
          if (has[k] && live) {
            Pack<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float xh = (vx[a][k].get(i) - mean[a]) * rstd[a];
              o.set(i, rstd[a] * (gz[k][i] * wv[k][i] - fmaf(xh, s2, s1)));
            }
            *reinterpret_cast<Pack<T, VEC>*>(dx + b * s.N * s.C + out[k]) = o;
          }
      }
    }
  }
  if (!parts) return;
  // the rows of a sample share channels: a row of the buffer for each of them and each of the block's samples
  parts += static_cast<int64_t>(blockIdx.x) * 2 * s.C;
  const int V = s.G * across, rows = p.rows * static_cast<int>(s.N);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
      if (has[k]) {
        const int e = k * p.lanes + l, at = (r * static_cast<int>(s.N) + e / across) * V + g * across + e % across;
#pragma unroll
        for (int i = 0; i < VEC; ++i) buffer[at * VEC + i] = which ? acc_b[k][i] : acc_a[k][i];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < s.C; c += blockDim.x) {
      double sum = 0.0;
      for (int k = 0; k < rows; ++k) sum += buffer[k * V * VEC + c];
      parts[which * s.C + c] = static_cast<float>(sum);
    }
  }
}

enum Mode { kFused, kSums, kApply };

// Tiles: a block's chunk of a slab in registers; blocks keep their slab (and chunk, where fused) and walk the samples.
// between: (B, chunks, G) pairs s1, s2 between the two kernels of samples that no cluster holds.
template <typename T, typename U, int ACT, int VEC, int MODE>
__global__ void __launch_bounds__(kMaxThreads) tiles_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                            const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                            const float* __restrict__ bias, T* __restrict__ dx, float* parts,
                                                            const Shape s, const Plan p, float2* between) {
  constexpr int kK = sizeof(T) == 4 ? 8 : 4;
  __shared__ float part[kMaxThreads];
  __shared__ float first[kMaxThreads], second[kMaxThreads];
  __shared__ float2 mine[kMaxThreads];
  __shared__ float buffer[kMaxThreads * VEC];
  const int cg = s.C / s.G, across = cg / VEC, groups = p.slab / cg;
  const int v = threadIdx.x % p.V, r = threadIdx.x / p.V, lanes = blockDim.x / p.V;
  // fused: clusters of chunks, slab fastest; else blocks, slab fastest, walking samples and chunks
  const int per_team = MODE == kFused ? p.chunks : 1;
  const int team = blockIdx.x / per_team, slab = team % p.slabs, first_work = team / p.slabs;
  const int teams = gridDim.x / per_team / p.slabs;
  const int c = slab * p.slab + v * VEC, j = v / across, g = slab * groups + j;
  const bool there = r < lanes && c < s.C;
  float wv[VEC], bv[VEC], acc_a[VEC], acc_b[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    wv[i] = there && w ? __ldg(w + c + i) : 1.0f;
    bv[i] = there && bias ? __ldg(bias + c + i) : 0.0f;
    acc_a[i] = acc_b[i] = 0.0f;
  }
  const float per = 1.0f / (static_cast<float>(s.N) * static_cast<float>(cg));
  const int64_t works = MODE == kFused ? s.B : s.B * p.chunks;
  for (int64_t at = first_work; at < works; at += teams) {
    const int64_t work = MODE == kApply ? works - 1 - at : at;      // what the other kernel read last is read first
    const int64_t b = MODE == kFused ? work : work / p.chunks;
    const int chunk = static_cast<int>(MODE == kFused ? blockIdx.x % p.chunks : work % p.chunks);
    const int row0 = chunk * p.chunk_rows, rows = min(p.chunk_rows, static_cast<int>(s.N) - row0);
    const float mean = there ? mean_in[b * s.G + g] : 0.0f, rstd = there ? rstd_in[b * s.G + g] : 0.0f;
    Pack<T, VEC> vx[kK];
    float gz[kK][VEC];
    {
      Pack<U, VEC> vg[kK];
      const T* from = x + b * s.x_sample + (row0 + r) * s.x_row + c;
      const U* from_g = gy + b * s.g_sample + (row0 + r) * s.g_row + c;
#pragma unroll
      for (int k = 0; k < kK; ++k)
        if (there && r + k * lanes < rows) {
          vx[k] = *reinterpret_cast<const Pack<T, VEC>*>(from + k * lanes * s.x_row);
          vg[k] = *reinterpret_cast<const Pack<U, VEC>*>(from_g + k * lanes * s.g_row);
        }
#pragma unroll
      for (int k = 0; k < kK; ++k)
        if (there && r + k * lanes < rows) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) gz[k][i] = vg[k].get(i);
        }
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < kK; ++k)
      if (there && r + k * lanes < rows) {
        float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = (vx[k].get(i) - mean) * rstd;
          gz[k][i] *= slope<ACT>(fmaf(wv[i], xh, bv[i]));
          if (MODE != kApply) {
            acc_a[i] += gz[k][i];
            acc_b[i] = fmaf(gz[k][i], xh, acc_b[i]);
            const float t = gz[k][i] * wv[i];
            t1 += t;
            t2 = fmaf(t, xh, t2);
          }
        }
        s1 += t1, s2 += t2;
      }
    if constexpr (MODE != kApply) {
      group_sums(s1, p.V, lanes, across, groups, part, first);
      group_sums(s2, p.V, lanes, across, groups, part, second);
      if (MODE == kSums) {
        if (there && r == 0 && v % across == 0) between[(b * p.chunks + chunk) * s.G + g] = make_float2(first[j], second[j]);
        __syncthreads();
        continue;
      }
      if (p.chunks > 1) {
        for (int k = threadIdx.x; k < groups; k += blockDim.x) mine[k] = make_float2(first[k], second[k]);
        cg_::cluster_group cluster = cg_::this_cluster();
        cluster.sync();
        for (int k = threadIdx.x; k < groups; k += blockDim.x) {
          float t1 = 0.0f, t2 = 0.0f;
          for (int q = 0; q < p.chunks; ++q) {
            const float2 t = cluster.map_shared_rank(mine, q)[k];
            t1 += t.x, t2 += t.y;
          }
          first[k] = t1, second[k] = t2;
        }
        cluster.sync();                            // every block has read the others' parts
      }
    } else {
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      for (int k = warp; k < groups && slab * groups + k < s.G; k += warps) {
        const float2* f = between + b * p.chunks * s.G + slab * groups + k;
        float t1 = 0.0f, t2 = 0.0f;
        for (int q = lane; q < p.chunks; q += 32) {
          const float2 t = f[static_cast<int64_t>(q) * s.G];
          t1 += t.x, t2 += t.y;
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) {
          t1 += __shfl_xor_sync(0xffffffffu, t1, m);
          t2 += __shfl_xor_sync(0xffffffffu, t2, m);
        }
        if (lane == 0) first[k] = t1, second[k] = t2;
      }
      __syncthreads();
    }
    if constexpr (MODE != kSums) {
      if (dx && there) {
        const float m1 = first[j] * per, m2 = second[j] * per;
        T* to = dx + (b * s.N + row0 + r) * s.C + c;
#pragma unroll
        for (int k = 0; k < kK; ++k)
          if (r + k * lanes < rows) {
            Pack<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float xh = (vx[k].get(i) - mean) * rstd;
              o.set(i, rstd * (gz[k][i] * wv[i] - fmaf(xh, m2, m1)));
            }
            *reinterpret_cast<Pack<T, VEC>*>(to + static_cast<int64_t>(k) * lanes * s.C) = o;
          }
      }
      __syncthreads();                             // first and second are this work's until here
    }
  }
  if (MODE != kApply && parts) {
    const int64_t row = MODE == kFused ? static_cast<int64_t>(first_work) * p.chunks + blockIdx.x % p.chunks : first_work;
    channel_sums<VEC>(acc_a, acc_b, v, p.V, r, lanes, c, s.C, there, buffer, parts + row * 2 * s.C);
  }
}

// dw and db from the blocks' parts: a warp takes 32 neighbouring columns' parts w, w + 8, ..., the warps' sums join in order
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ parts, int64_t n, int C, float* __restrict__ dw,
                                                   float* __restrict__ db) {
  __shared__ double sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
  double sum = 0.0;
  if (column < 2 * C)
    for (int64_t k = warp; k < n; k += 8) sum += parts[k * 2 * C + column];
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && column < 2 * C) {
    for (int k = 1; k < 8; ++k) sum += sums[k][lane];
    if (column < C) {
      if (db) db[column] = static_cast<float>(sum);
    } else if (dw) {
      dw[column - C] = static_cast<float>(sum);
    }
  }
}

// the sum over the block, in every thread; red: 8 floats
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += red[w];
  __syncthreads();
  return s;
}

// Wide groups: a block per sample and group, in two passes
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(256) wide_kernel(const U* __restrict__ gy, const T* __restrict__ x, const float* __restrict__ mean_in,
                                                   const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                   const float* __restrict__ bias, T* __restrict__ dx, const Shape s) {
  __shared__ float red[8];
  const int cg = s.C / s.G;
  const int64_t n = s.N * cg;
  for (int64_t at = blockIdx.x; at < s.B * s.G; at += gridDim.x) {
    const int64_t b = at / s.G;
    const int c0 = static_cast<int>(at % s.G) * cg;
    const float mean = mean_in[at], rstd = rstd_in[at];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
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
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float wc = w ? w[c] : 1.0f;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      const float a = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope<ACT>(fmaf(wc, xh, bias ? bias[c] : 0.0f)) * wc;
      store_f32(dx + (b * s.N + r) * s.C + c, rstd * (a - fmaf(xh, s2, s1)));
    }
  }
}

// Wide groups: a thread per channel walks a share of the rows, into the parts that join_kernel adds
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(256) wide_channels_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                            const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, const float* __restrict__ w,
                                                            const float* __restrict__ bias, float* __restrict__ parts, const Shape s) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= s.C) return;
  const int g = c / (s.C / s.G);
  const float wc = w ? w[c] : 1.0f, bc = bias ? bias[c] : 0.0f;
  double a = 0.0, d = 0.0;
  for (int64_t i = blockIdx.y; i < s.B * s.N; i += gridDim.y) {
    const int64_t b = i / s.N, r = i % s.N;
    const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean_in[b * s.G + g]) * rstd_in[b * s.G + g];
    const float gz = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope<ACT>(fmaf(wc, xh, bc));
    a += gz;
    d += static_cast<double>(gz) * xh;
  }
  parts[static_cast<int64_t>(blockIdx.y) * 2 * s.C + c] = static_cast<float>(a);
  parts[static_cast<int64_t>(blockIdx.y) * 2 * s.C + s.C + c] = static_cast<float>(d);
}

Plan plan_of(const Shape& s, int size, bool aligned) { return make_plan(s, size, backward_rows(size), num_sms(), aligned); }

// Blocks that walk the samples: as many as are resident, two of 512 threads per SM at most
int64_t walkers(const Shape& s, const Plan& p) {
  const int64_t resident = static_cast<int64_t>(num_sms()) * std::max(1, std::min(4, 640 / p.threads));
  if (p.kind == kUnits) return std::min(resident, (s.B + p.rows - 1) / p.rows);
  if (p.kind == kWide) return std::min<int64_t>(s.B * s.N, 32);
  // per slab: teams of a cluster, or blocks
  const int64_t team = p.fused ? p.chunks : 1;
  return std::max<int64_t>(1, std::min(p.fused ? s.B : s.B * p.chunks, resident / (p.slabs * team))) * team;
}

}  // namespace

size_t backward_workspace(const Shape& s, int size) {
  size_t bytes = 16;
  for (bool aligned : {false, true}) {
    const Plan p = plan_of(s, size, aligned);
    size_t parts = sizeof(float) * 2 * static_cast<size_t>(s.C) * walkers(s, p);
    parts = (parts + 15) / 16 * 16;
    if (p.kind == kTiles && !p.fused) parts += sizeof(float2) * static_cast<size_t>(s.B) * p.chunks * s.G;
    bytes = std::max(bytes, parts);
  }
  return bytes;
}

namespace {

template <typename T, typename U, int ACT, int VEC>
int run(const U* gy, const T* x, const float* mean, const float* rstd, const float* w, const float* bias, T* dx, bool want_parts,
        const Shape& s, const Plan& p, void* ws, cudaStream_t st) {
  const char* what = "group_norm backward";
  const int64_t n = walkers(s, p);
  float* parts = want_parts ? static_cast<float*>(ws) : nullptr;
  if (p.kind == kUnits) {
    const int smem = p.rows * static_cast<int>(s.N) * s.C * static_cast<int>(sizeof(float));
    const void* fn = p.slots == 1 ? reinterpret_cast<const void*>(&units_kernel<T, U, ACT, VEC, 1>)
                                  : reinterpret_cast<const void*>(&units_kernel<T, U, ACT, VEC, 4>);
    if (smem > 48 * 1024)
      if (int e = allow_smem(fn, smem)) return e;
    const unsigned grid = static_cast<unsigned>(n);
    if (p.slots == 1) units_kernel<T, U, ACT, VEC, 1><<<grid, p.threads, smem, st>>>(gy, x, mean, rstd, w, bias, dx, parts, s, p);
    else units_kernel<T, U, ACT, VEC, 4><<<grid, p.threads, smem, st>>>(gy, x, mean, rstd, w, bias, dx, parts, s, p);
    return launched(what);
  }
  float2* between = reinterpret_cast<float2*>(static_cast<char*>(ws) + (sizeof(float) * 2 * s.C * n + 15) / 16 * 16);
  Shape shape = s;
  Plan plan = p;
  void* args[] = {&gy, &x, &mean, &rstd, &w, &bias, &dx, &parts, &shape, &plan, &between};
  const unsigned grid = static_cast<unsigned>(n * p.slabs);
  if (p.fused) return launch(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kFused>), grid, p.threads, p.chunks, st, args, what);
  if (int e = launch(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kSums>), grid, p.threads, 1, st, args, what)) return e;
  if (!dx) return 0;
  return launch(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kApply>), grid, p.threads, 1, st, args, what);
}

}  // namespace

size_t forward_workspace(const Shape& s, int size);

}  // namespace gn
}  // namespace bpc

using namespace bpc;
using namespace bpc::gn;

extern "C" size_t bpc_group_norm_workspace_size(int64_t B, int64_t N, int32_t C, int32_t G, int32_t x_dtype, int32_t backward) {
  const Shape s{B, N, C, G, 0, 0, 0, 0};
  if (B < 1 || N < 1 || !size_of(x_dtype) || check_shape(s, BPC_ACT_NONE, x_dtype, x_dtype, "group_norm")) return 0;
  return backward ? backward_workspace(s, size_of(x_dtype)) : forward_workspace(s, size_of(x_dtype));
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
  const int size = size_of(x_dtype), y_size = size_of(y_dtype);
  if (!aligned(x, size) || !aligned(dx, size) || !aligned(gy, y_size) || !aligned(mean, 4) || !aligned(rstd, 4) ||
      !aligned(weight, 4) || !aligned(bias, 4) || !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "group_norm backward: buffer not aligned to its type (workspace: 16 bytes)");
  if (workspace_bytes < bpc_group_norm_workspace_size(B, N, C, G, x_dtype, 1))
    return fail(BPC_ERR_SPACE, "group_norm backward: workspace too small");
  if (!dx && !dw && !db) return 0;
  // gy's accesses are as many elements as x's: 8 bytes of 16-bit gradients of fp32 features
  const bool whole = aligned(x, 16) && aligned(dx, 16) && aligned(gy, 16) && x_sample_stride * size % 16 == 0 &&
                     x_row_stride * size % 16 == 0 && gy_sample_stride * y_size % 16 == 0 && gy_row_stride * y_size % 16 == 0;
  const Plan p = plan_of(s, size, whole);
  const bool want = dw || db;
  const int e = with_types(x_dtype, y_dtype, [&](auto xt, auto yt) {
    return with_act(activation, [&](auto act) {
      typedef typename decltype(xt)::type T;
      typedef typename decltype(yt)::type U;
      constexpr int ACT = decltype(act)::value;
      const U* g = static_cast<const U*>(gy);
      const T* from = static_cast<const T*>(x);
      T* to = static_cast<T*>(dx);
      if (p.kind == kWide) {
        if (dx) {
          const unsigned grid = static_cast<unsigned>(std::min<int64_t>(B * G, 8 * num_sms()));
          wide_kernel<T, U, ACT><<<grid, 256, 0, st>>>(g, from, mean, rstd, weight, bias, to, s);
          if (int e = launched(what)) return e;
        }
        if (!want) return 0;
        const dim3 grid((C + 255) / 256, static_cast<unsigned>(walkers(s, p)));
        wide_channels_kernel<T, U, ACT><<<grid, 256, 0, st>>>(g, from, mean, rstd, weight, bias, static_cast<float*>(workspace), s);
        return launched(what);
      }
      if (p.vec == 1) return run<T, U, ACT, 1>(g, from, mean, rstd, weight, bias, to, want, s, p, workspace, st);
      return run<T, U, ACT, 16 / sizeof(T)>(g, from, mean, rstd, weight, bias, to, want, s, p, workspace, st);
    });
  });
  if (e || !want) return e;
  join_kernel<<<(2 * C + 31) / 32, 256, 0, st>>>(static_cast<const float*>(workspace), walkers(s, p), C, dw, db);
  return launched(what);
}
