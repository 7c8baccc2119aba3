// Group normalisation with an activation over channels-last features: the gradients.
//
//   gz = gy act'(z), A_c = sum_n gz, B_c = sum_n gz xh over a sample, s1 = sum_c w_c A_c, s2 = sum_c w_c B_c over its
//   group (z, xh as in the forward pass):
//     dx = rstd (gz w_c - (s1 + xh s2) / (N C / G));   dw_c = sum_b B_c;   db_c = sum_b A_c
//
// One read of gy and x and one write of dx where a sample's slab fits the registers of a block or a cluster.  A thread
// always has the same channels and walks the samples, so that dw and db are sums in registers until the end: a part per
// block, joined in order in fp64 (deterministic, no atomics).
//   512 x 504 x 512 fp32 with bf16 gradients: 289 us, 4.6 TB/s of 1.32 GB; 1.36 M samples of 96 bf16 channels: 189 us, 4.2 TB/s of
// 794 MB, bound by instructions (32 a value, of which the activation's are 5).
#include "group_norm.cuh"

namespace bpc {
namespace gn {
namespace {

namespace cg_ = cooperative_groups;

// The channels' sums of a block: thread (row r, vector v) has VEC channels from c on, `rows` rows of threads; into
// parts[block][2][C]
template <int VEC>
__device__ __forceinline__ void channel_sums(const uint64_t (&a)[(VEC + 1) / 2], const uint64_t (&d)[(VEC + 1) / 2], int v, int V, int r,
                                             int rows, int c, int C, bool there, float* buffer, float* parts) {
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (there) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const uint64_t x = which ? d[i / 2] : a[i / 2];
        buffer[(r * V + v) * VEC + i] = i % 2 ? f2_hi(x) : f2_lo(x);
      }
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

// Units: a sample's group per `lanes` lanes, SLOTS vectors each; a thread's slots are the same places of every sample, and
// the next samples' are on their way while one is worked on.
template <typename T, typename U, int ACT, int VEC, int SLOTS>
__global__ void __launch_bounds__(kUnitThreads) units_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                             const float2* __restrict__ stats,
                                                             const float* __restrict__ w, const float* __restrict__ bias, T* __restrict__ dx,
                                                             float* parts,
                                                             const Shape s, const Plan p) {
  constexpr int kP = Pack<T, VEC>::kPairs;
  extern __shared__ __align__(16) uint8_t smem[];
  const int cg = s.C / s.G, across = cg / VEC;
  const int unit = threadIdx.x / p.lanes, l = threadIdx.x % p.lanes;
  const int g = unit % s.G, r = unit / s.G;
  const bool there = r < p.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * p.rows, b0 = static_cast<int64_t>(blockIdx.x) * p.rows;
  const int rounds = static_cast<int>((s.B - b0 + step - 1) / step);                          // of the block
  const int mine = there && b0 + r < s.B ? static_cast<int>((s.B - b0 - r + step - 1) / step) : 0;
  const T* from[SLOTS];
  const U* from_g[SLOTS];
  T* to[SLOTS];
  bool has[SLOTS];
  uint64_t wv[SLOTS][kP], bv[SLOTS][kP], acc_a[SLOTS][kP], acc_b[SLOTS][kP];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    const int e = k * p.lanes + l, row = e / across, c = g * cg + e % across * VEC;
    has[k] = there && row < s.N;
    from[k] = x + (b0 + r) * s.x_sample + row * s.x_row + c;
    from_g[k] = gy + (b0 + r) * s.g_sample + row * s.g_row + c;
    to[k] = dx + ((b0 + r) * s.N + row) * s.C + c;
    channels<VEC>(w, c, has[k], 1.0f, wv[k]);
    channels<VEC>(bias, c, has[k], 0.0f, bv[k]);
#pragma unroll
    for (int i = 0; i < kP; ++i) acc_a[k][i] = acc_b[k][i] = 0;
  }
  const float per = 1.0f / (static_cast<float>(s.N) * static_cast<float>(cg));
  const int64_t x_step = step * s.x_sample, g_step = step * s.g_sample, o_step = step * s.N * s.C;
  // a stage: the block's vectors of x, those of gy, the statistics; a thread's places in it, and the stages of the sample
  // fetched and of the one worked on
  using X = Copied<T, VEC>;
  using Y = Copied<U, VEC>;
  constexpr int kDepth = units_depth(units_bytes(X::kBytes, Y::kBytes, SLOTS, true));
  const uint32_t x_bytes = blockDim.x * X::kBytes, g_bytes = blockDim.x * Y::kBytes;
  const uint32_t at_x = threadIdx.x * X::kBytes, at_g = SLOTS * x_bytes + threadIdx.x * Y::kBytes;
  const uint32_t at_stat = SLOTS * (x_bytes + g_bytes) + threadIdx.x * 8, stage_bytes = SLOTS * (x_bytes + g_bytes) + blockDim.x * 8;
  const uint32_t base = smem_u32(smem);
  uint32_t fetched = 0, used = 0;
  const float2* stat = stats + (b0 + r) * s.G + g;
  const int64_t stat_step = step * s.G;
  auto fetch = [&](int round) {
    if (round < mine) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(base + fetched + at_stat), "l"(stat) : "memory");
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (has[k]) {
          X::fetch(base + fetched + at_x + k * x_bytes, from[k]);
          Y::fetch(base + fetched + at_g + k * g_bytes, from_g[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) from[k] += x_step, from_g[k] += g_step;
    stat += stat_step;
    fetched = fetched == (kDepth - 1) * stage_bytes ? 0 : fetched + stage_bytes;
    cp_commit();
  };
#pragma unroll
  for (int round = 0; round < kDepth - 1; ++round) fetch(round);
  for (int round = 0; round < rounds; ++round) {
    fetch(round + kDepth - 1);
    cp_wait<kDepth - 1>();
    const bool live = round < mine;
    const float2 f = *reinterpret_cast<const float2*>(smem + used + at_stat);
    const float mean = live ? f.x : 0.0f, rstd = live ? f.y : 0.0f;
    const uint64_t scale = f2_of(rstd), minus = f2_of(-mean);
    uint64_t xh[SLOTS][kP], gz[SLOTS][kP], s1 = 0, s2 = 0;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      Pack<T, VEC> vx = Pack<T, VEC>();            // zeros: nothing to any sum
      Pack<U, VEC> vg = Pack<U, VEC>();
      if (X::kCopies && Y::kCopies) {              // what was not fetched is replaced, not asked for: nearly all is
        vx = X::take(smem, used + at_x + k * x_bytes, nullptr), vg = Y::take(smem, used + at_g + k * g_bytes, nullptr);
        if (!(has[k] && live)) vx = Pack<T, VEC>(), vg = Pack<U, VEC>();
      } else if (has[k] && live) {                 // the pointers are kDepth samples ahead
        vx = X::take(smem, used + at_x + k * x_bytes, from[k] - kDepth * x_step);
        vg = Y::take(smem, used + at_g + k * g_bytes, from_g[k] - kDepth * g_step);
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        xh[k][i] = f2_mul(f2_add(vx.pair(i), minus), scale);
        gz[k][i] = vg.pair(i);
      }
    }
    used = used == (kDepth - 1) * stage_bytes ? 0 : used + stage_bytes;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        gz[k][i] = f2_mul(gz[k][i], slope<ACT>(f2_fma(wv[k][i], xh[k][i], bv[k][i])));
        acc_a[k][i] = f2_add(acc_a[k][i], gz[k][i]);
        acc_b[k][i] = f2_fma(gz[k][i], xh[k][i], acc_b[k][i]);
        gz[k][i] = f2_mul(gz[k][i], wv[k][i]);
        s1 = f2_add(s1, gz[k][i]);
        s2 = f2_fma(gz[k][i], xh[k][i], s2);
      }
    const float m1 = lanes_sum(both<VEC>(s1), p.lanes), m2 = lanes_sum(both<VEC>(s2), p.lanes);
    if (dx) {
      const uint64_t u1 = f2_of(-m1 * per), u2 = f2_of(-m2 * per);
#pragma unroll
      for (int k = 0; k < SLOTS; ++k) {
        Pack<T, VEC> o;
#pragma unroll
        for (int i = 0; i < kP; ++i) o.set(i, f2_mul(scale, f2_add(gz[k][i], f2_fma(xh[k][i], u2, u1))));
        if (has[k] && live) *reinterpret_cast<Pack<T, VEC>*>(to[k]) = o;
        to[k] += o_step;
      }
    }
  }
  if (!parts) return;
  // every copy has been taken: its memory holds the channels' sums now.  The rows of a sample share channels: a row of the
  // buffer for each of them and each of the block's samples
  parts += static_cast<int64_t>(blockIdx.x) * 2 * s.C;
  float* buffer = reinterpret_cast<float*>(smem);
  const int V = s.G * across, rows = p.rows * static_cast<int>(s.N);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
      if (has[k]) {
        const int e = k * p.lanes + l, at = (r * static_cast<int>(s.N) + e / across) * V + g * across + e % across;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const uint64_t t = which ? acc_b[k][i / 2] : acc_a[k][i / 2];
          buffer[at * VEC + i] = i % 2 ? f2_hi(t) : f2_lo(t);
        }
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

// Tiles: a block's chunk of a slab in registers, the next sample's on its way meanwhile; blocks keep their slab and chunk and
// walk the samples.  between: (B, chunks, G) pairs s1, s2 between the two kernels of samples that no cluster holds.
template <typename T, typename U, int ACT, int VEC, int MODE>
__global__ void __launch_bounds__(kTileThreads, 2) tiles_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                            const float2* __restrict__ stats,
                                                            const float* __restrict__ w, const float* __restrict__ bias, T* __restrict__ dx,
                                                            float* parts,
                                                            const Shape s, const Plan p, float2* between) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float part[2][2 * kTileThreads];
  __shared__ float2 mine[kTileThreads];
  const int cg = s.C / s.G, across = cg / VEC, groups = p.slab / cg;
  const int v = threadIdx.x % p.V, r = threadIdx.x / p.V, lanes = blockDim.x / p.V, j = v / across;
  // what the other kernel read last is read first
  const int chunk0 = blockIdx.x % p.chunks, slab = blockIdx.x / p.chunks, chunk = MODE == kApply ? p.chunks - 1 - chunk0 : chunk0;
  const int c = slab * p.slab + v * VEC, g = slab * groups + j;
  const int row0 = chunk * p.chunk_rows, rows = min(p.chunk_rows, static_cast<int>(s.N) - row0);
  const bool there = r < lanes && c < s.C, speaks = there && r == 0 && v % across == 0;
  const int n = there && r < rows ? (rows - r + lanes - 1) / lanes : 0;        // this thread's rows
  auto sample = [&](int64_t k) { return MODE == kApply ? s.B - 1 - k : k; };
  const T* from = x + static_cast<int64_t>(row0 + r) * s.x_row + c;
  const U* from_g = gy + static_cast<int64_t>(row0 + r) * s.g_row + c;
  T* to = dx + static_cast<int64_t>(row0 + r) * s.C + c;
  const int64_t x_step = lanes * s.x_row, g_step = lanes * s.g_row, o_step = static_cast<int64_t>(lanes) * s.C;
  Ahead<T, VEC, kRows> ahead_x(smem);
  Ahead<U, VEC, kRows> ahead_g(smem + Ahead<T, VEC, kRows>::kBytes * kTileThreads);
  float2 next = make_float2(0.0f, 0.0f);
  auto fetch = [&](int64_t b) {
    ahead_x.fetch(from + b * s.x_sample, x_step, n);
    ahead_g.fetch(from_g + b * s.g_sample, g_step, n);
    if (there) next = stats[b * s.G + g];
  };
  fetch(sample(blockIdx.y));
  constexpr int kP = Pack<T, VEC>::kPairs;
  uint64_t wv[kP], bv[kP], acc_a[kP], acc_b[kP];
  channels<VEC>(w, c, there, 1.0f, wv);
  channels<VEC>(bias, c, there, 0.0f, bv);
#pragma unroll
  for (int i = 0; i < kP; ++i) acc_a[i] = acc_b[i] = 0;
  const float per = 1.0f / (static_cast<float>(s.N) * static_cast<float>(cg));
  int turn = 0;
  for (int64_t at = blockIdx.y; at < s.B; at += gridDim.y) {
    const int64_t b = sample(at);
    const uint64_t scale = f2_of(next.y), minus = f2_of(-next.x);
    Pack<T, VEC> vx[kRows];
    uint64_t gz[kRows][kP];
    float sums[2] = {0.0f, 0.0f};
    cp_wait_all();
    ahead_x.take(vx);
    {
      Pack<U, VEC> vg[kRows];
      ahead_g.take(vg);
      uint64_t a[kP], d[kP];
#pragma unroll
      for (int i = 0; i < kP; ++i) a[i] = d[i] = 0;
      with_rows(n == kRows, [&](auto all) {
#pragma unroll
        for (int k = 0; k < kRows; ++k)
          if (decltype(all)::value || k < n) {
#pragma unroll
            for (int i = 0; i < kP; ++i) {
              const uint64_t xh = f2_mul(f2_add(vx[k].pair(i), minus), scale);
              gz[k][i] = f2_mul(vg[k].pair(i), slope<ACT>(f2_fma(wv[i], xh, bv[i])));
              if (MODE != kApply) {
                a[i] = f2_add(a[i], gz[k][i]);
                d[i] = f2_fma(gz[k][i], xh, d[i]);
              }
            }
          }
      });
      if constexpr (MODE != kApply) {
        // the channels' sums of this sample, weighed, are the group's
        uint64_t t1 = 0, t2 = 0;
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          acc_a[i] = f2_add(acc_a[i], a[i]);
          acc_b[i] = f2_add(acc_b[i], d[i]);
          t1 = f2_fma(a[i], wv[i], t1);
          t2 = f2_fma(d[i], wv[i], t2);
        }
        sums[0] = both<VEC>(t1), sums[1] = both<VEC>(t2);
      }
    }
    if (at + gridDim.y < s.B) fetch(sample(at + gridDim.y));
    if constexpr (MODE != kApply) {
      // two buffers in turn: a sample has one barrier
      group_sums(sums, p.V, lanes, across, v, part[turn]);
      turn ^= 1;
      if (MODE == kSums) {
        if (speaks) between[(b * p.chunks + chunk) * s.G + g] = make_float2(sums[0], sums[1]);
        continue;
      }
      if (p.chunks > 1) {
        if (speaks) mine[j] = make_float2(sums[0], sums[1]);
        cg_::cluster_group cluster = cg_::this_cluster();
        cluster.sync();
        sums[0] = sums[1] = 0.0f;
        for (int q = 0; q < p.chunks; ++q) {
          const float2 t = cluster.map_shared_rank(mine, q)[j];
          sums[0] += t.x, sums[1] += t.y;
        }
        cluster.sync();                            // every block has read the others' parts
      }
    } else {
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      __syncthreads();
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
        if (lane == 0) mine[k] = make_float2(t1, t2);
      }
      __syncthreads();
      sums[0] = mine[j].x, sums[1] = mine[j].y;
    }
    if constexpr (MODE != kSums) {
      if (dx) {
        const uint64_t u1 = f2_of(-sums[0] * per), u2 = f2_of(-sums[1] * per);
        T* out = to + b * s.N * s.C;
        with_rows(n == kRows, [&](auto all) {
#pragma unroll
          for (int k = 0; k < kRows; ++k) {
            if (decltype(all)::value || k < n) {
              Pack<T, VEC> o;
#pragma unroll
              for (int i = 0; i < kP; ++i) {
                const uint64_t xh = f2_mul(f2_add(vx[k].pair(i), minus), scale);
                o.set(i, f2_mul(scale, f2_fma(gz[k][i], wv[i], f2_fma(xh, u2, u1))));
              }
              *reinterpret_cast<Pack<T, VEC>*>(out) = o;
            }
            out += o_step;
          }
        });
      }
    }
  }
  if (MODE != kApply && parts) {
    // the copies have all been taken: their memory holds the channels' sums now (VEC floats a thread are no more than them)
    float* buffer = reinterpret_cast<float*>(smem);
    channel_sums<VEC>(acc_a, acc_b, v, p.V, r, lanes, c, s.C, there, buffer,
                      parts + (static_cast<int64_t>(blockIdx.y) * p.chunks + chunk) * 2 * s.C);
  }
}

// dw and db from the blocks' parts: a warp takes 32 neighbouring columns' parts w, w + 32, ..., the warps' sums join in order
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ parts, int64_t n, int C, float* __restrict__ dw,
                                                    float* __restrict__ db) {
  __shared__ double sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
  double sum = 0.0;
  if (column < 2 * C) {
#pragma unroll 8
    for (int64_t k = warp; k < n; k += 32) sum += parts[k * 2 * C + column];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  // a warp per column
  sum = sums[lane][warp];
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < 2 * C) {
    if (mine < C) {
      if (db) db[mine] = static_cast<float>(sum);
    } else if (dw) {
      dw[mine - C] = static_cast<float>(sum);
    }
  }
}

// Wide groups: a block per sample and group, in two passes
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(256) wide_kernel(const U* __restrict__ gy, const T* __restrict__ x, const float2* __restrict__ stats,
                                                   const float* __restrict__ w, const float* __restrict__ bias, T* __restrict__ dx,
                                                   const Shape s) {
  __shared__ double red[8];
  const int cg = s.C / s.G;
  const int64_t n = s.N * cg;
  for (int64_t at = blockIdx.x; at < s.B * s.G; at += gridDim.x) {
    const int64_t b = at / s.G;
    const int c0 = static_cast<int>(at % s.G) * cg;
    const float mean = stats[at].x, rstd = stats[at].y;
    double sum1 = 0.0, sum2 = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float wc = w ? w[c] : 1.0f;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      const float a = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope1<ACT>(fmaf(wc, xh, bias ? bias[c] : 0.0f)) * wc;
      sum1 += a;
      sum2 = fma(static_cast<double>(a), static_cast<double>(xh), sum2);
    }
    const float s1 = block_mean(sum1, n, red), s2 = block_mean(sum2, n, red);
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float wc = w ? w[c] : 1.0f;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      const float a = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope1<ACT>(fmaf(wc, xh, bias ? bias[c] : 0.0f)) * wc;
      store_f32(dx + (b * s.N + r) * s.C + c, rstd * (a - fmaf(xh, s2, s1)));
    }
  }
}

// Wide groups: a thread per channel walks a share of the rows, into the parts that join_kernel adds
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(256) wide_channels_kernel(const U* __restrict__ gy, const T* __restrict__ x,
                                                            const float2* __restrict__ stats,
                                                            const float* __restrict__ w, const float* __restrict__ bias, float* __restrict__ parts,
                                                            const Shape s) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= s.C) return;
  const int g = c / (s.C / s.G);
  const float wc = w ? w[c] : 1.0f, bc = bias ? bias[c] : 0.0f;
  double a = 0.0, d = 0.0;
  for (int64_t i = blockIdx.y; i < s.B * s.N; i += gridDim.y) {
    const int64_t b = i / s.N, r = i % s.N;
    const float2 f = stats[b * s.G + g];
    const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - f.x) * f.y;
    const float gz = load_f32(gy + b * s.g_sample + r * s.g_row + c) * slope1<ACT>(fmaf(wc, xh, bc));
    a += gz;
    d += static_cast<double>(gz) * xh;
  }
  parts[static_cast<int64_t>(blockIdx.y) * 2 * s.C + c] = static_cast<float>(a);
  parts[static_cast<int64_t>(blockIdx.y) * 2 * s.C + s.C + c] = static_cast<float>(d);
}

Plan plan_of(const Shape& s, int size, bool aligned) { return make_plan(s, size, num_sms(), aligned, true); }

constexpr int kTilesPerSm = 2;
// Samples whose gradients a thread adds up in fp32 before they are joined in fp64.  Values that are all alike round the same way:
// 3,333 times 0.1 is 560 roundings of 2^-24 off, 256 times 40.
constexpr int64_t kWalk = 256;

// Parts of dw and db: one per block that walks the samples, per slab
int64_t parts_of(const Shape& s, const Plan& p) {
  if (p.kind == kUnits) {
    const int64_t blocks = (s.B + p.rows - 1) / p.rows;
    return std::min(blocks, std::max(static_cast<int64_t>(num_sms()) * std::max(1, 1024 / p.threads), (blocks + kWalk - 1) / kWalk));
  }
  if (p.kind == kWide) return std::min<int64_t>(s.B * s.N, 32);
  return static_cast<int64_t>(tiles_grid(s, p, kTilesPerSm, num_sms(), kWalk).y) * p.chunks;
}

}  // namespace

size_t backward_workspace(const Shape& s, int size) {
  size_t bytes = 16;
  for (bool aligned : {false, true}) {
    const Plan p = plan_of(s, size, aligned);
    size_t parts = sizeof(float) * 2 * static_cast<size_t>(s.C) * parts_of(s, p);
    parts = (parts + 15) / 16 * 16;
    if (p.kind == kTiles && !p.fused) parts += sizeof(float2) * static_cast<size_t>(s.B) * p.chunks * s.G;
    bytes = std::max(bytes, parts);
  }
  return bytes;
}

namespace {

template <typename T, typename U, int ACT, int VEC, int SLOTS>
int run_units(const U* gy, const T* x, const float2* stats, const float* w, const float* bias, T* dx, float* parts, const Shape& s,
              const Plan& p, cudaStream_t st) {
  const int smem = units_smem(p, s, sizeof(T), sizeof(U), true);
  Shape shape = s;
  Plan plan = p;
  void* args[] = {&gy, &x, &stats, &w, &bias, &dx, &parts, &shape, &plan};
  return launch_clusters(reinterpret_cast<const void*>(&units_kernel<T, U, ACT, VEC, SLOTS>), dim3(static_cast<unsigned>(parts_of(s, p))),
                         dim3(p.threads), smem, st, args, 1, "group_norm backward");
}

template <typename T, typename U, int ACT, int VEC>
int run_tiles(const U* gy, const T* x, const float2* stats, const float* w, const float* bias, T* dx, float* parts, const Shape& s,
              const Plan& p, void* ws, cudaStream_t st) {
  const char* what = "group_norm backward";
  const int64_t n = parts_of(s, p);
  float2* between = reinterpret_cast<float2*>(static_cast<char*>(ws) + (sizeof(float) * 2 * s.C * n + 15) / 16 * 16);
  Shape shape = s;
  Plan plan = p;
  void* args[] = {&gy, &x, &stats, &w, &bias, &dx, &parts, &shape, &plan, &between};
  const int smem = std::max(Ahead<T, VEC, kRows>::kBytes + Ahead<U, VEC, kRows>::kBytes, VEC * static_cast<int>(sizeof(float))) * kTileThreads;
  const dim3 grid = tiles_grid(s, p, kTilesPerSm, num_sms(), kWalk);
  if (p.fused)
    return launch_clusters(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kFused>), grid, dim3(p.threads), smem, st, args, p.chunks, what);
  if (int e = launch_clusters(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kSums>), grid, dim3(p.threads), smem, st, args, 1, what)) return e;
  if (!dx) return 0;
  return launch_clusters(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kApply>), grid, dim3(p.threads), smem, st, args, 1, what);
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

extern "C" int bpc_group_norm_bwd(const void* gy, const void* x, const float* stats, const float* weight, const float* bias,
                                  void* dx, float* dw, float* db, int64_t B, int64_t N, int32_t C,
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
  if (!gy || !x || !stats || !workspace) return fail(BPC_ERR_ARG, "group_norm backward: null buffer");
  const int size = size_of(x_dtype), y_size = size_of(y_dtype);
  if (!aligned(x, size) || !aligned(dx, size) || !aligned(gy, y_size) || !aligned(stats, 8) ||
      !aligned(weight, 4) || !aligned(bias, 4) || !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "group_norm backward: buffer not aligned to its type (stats: 8 bytes, workspace: 16)");
  if (workspace_bytes < bpc_group_norm_workspace_size(B, N, C, G, x_dtype, 1))
    return fail(BPC_ERR_SPACE, "group_norm backward: workspace too small");
  if (!dx && !dw && !db) return 0;
  // accesses are of as many elements of gy as of x
  const int64_t full = 16 / size;
  auto whole_of = [&](const void* q, int64_t sample, int64_t row, int bytes) {
    return aligned(q, static_cast<int>(full) * bytes) && sample % full == 0 && row % full == 0;
  };
  const bool whole = whole_of(x, x_sample_stride, x_row_stride, size) && whole_of(dx, 0, 0, size) &&
                     whole_of(gy, gy_sample_stride, gy_row_stride, y_size);
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
      const float2* pairs = reinterpret_cast<const float2*>(stats);
      if (p.kind == kWide) {
        if (dx) {
          const unsigned grid = static_cast<unsigned>(std::min<int64_t>(B * G, 8 * num_sms()));
          wide_kernel<T, U, ACT><<<grid, 256, 0, st>>>(g, from, pairs, weight, bias, to, s);
          if (int e = launched(what)) return e;
        }
        if (!want) return 0;
        const dim3 grid((C + 255) / 256, static_cast<unsigned>(parts_of(s, p)));
        wide_channels_kernel<T, U, ACT><<<grid, 256, 0, st>>>(g, from, pairs, weight, bias, static_cast<float*>(workspace), s);
        return launched(what);
      }
      float* parts = want ? static_cast<float*>(workspace) : nullptr;
      if (p.kind == kUnits) {
        auto units = [&](auto vec, auto slots) {
          return run_units<T, U, ACT, decltype(vec)::value, decltype(slots)::value>(g, from, pairs, weight, bias, to, parts, s, p, st);
        };
        std::integral_constant<int, 1> one;
        std::integral_constant<int, 2> two;
        std::integral_constant<int, 4> four;
        if constexpr (sizeof(T) == 2)
          if (p.vec == 8) return units(std::integral_constant<int, 8>(), one);
        if (p.vec == 4) return p.slots == 1 ? units(four, one) : p.slots == 2 ? units(four, two) : units(four, four);
        return p.slots == 1 ? units(one, one) : p.slots == 2 ? units(one, two) : units(one, four);
      }
      if (p.vec == 1) return run_tiles<T, U, ACT, 1>(g, from, pairs, weight, bias, to, parts, s, p, workspace, st);
      return run_tiles<T, U, ACT, kTileVec>(g, from, pairs, weight, bias, to, parts, s, p, workspace, st);
    });
  });
  if (e || !want) return e;
  join_kernel<<<(2 * C + 31) / 32, 1024, 0, st>>>(static_cast<const float*>(workspace), parts_of(s, p), C, dw, db);
  return launched(what);
}
