// Group normalisation with an activation over channels-last features: the forward pass.
//
//   x (B, N, C), group g = channels [g C / G, (g + 1) C / G):  mean, var over the N C / G values of a sample and group
//   xh = (x - mean) rstd, rstd = 1 / sqrt(var + eps);   z = w_c xh + b_c;   y = act(z) = z s(u(z))
//     act: none (s = 1), SiLU (u = z), GELU in its tanh form (u = 2 sqrt(2 / pi) (z + 0.044715 z^3)), s the logistic
//     function
//
// One read of x and one write of y where a sample's slab fits the registers of a block or a cluster; the variance is the
// mean of the squared differences from the mean, never a difference of squares, and the parts of several blocks join as
// var n = sum (var_i n_i + n_i (mean_i - mean)^2).
//   512 x 504 x 512 fp32 into bf16 with 32 groups and SiLU: 158 us, 5.0 TB/s of 793 MB; 1.36 M samples of 96 bf16 channels in 3
// groups: 110 us, 4.8 TB/s.  Bound by instructions and the latency of the two joins of a sample as much as by memory: on
// pairs of values, with the rows that are all there told apart from those that are not, a tile takes half of what it took (34 -> 16 M
// instructions for 96 shots).  64 samples of 2,197 x 128 fp32 in one group each fit no cluster: 45 us with x read twice, the
// second time mostly from L2.
#include "group_norm.cuh"

namespace bpc {
namespace gn {
namespace {

namespace cg_ = cooperative_groups;

// Units: a sample's group per `lanes` lanes, SLOTS vectors each; a thread's slots are the same places of every sample, and
// the next samples' are on their way while one is worked on.
template <typename T, typename U, int ACT, int VEC, int SLOTS>
__global__ void __launch_bounds__(kUnitThreads) units_kernel(const T* __restrict__ x, U* __restrict__ y, float2* stats,
                                                             const float* __restrict__ w, const float* __restrict__ bias, const Shape s, const Plan p,
                                                             float eps) {
  constexpr int kP = Pack<T, VEC>::kPairs;
  const int cg = s.C / s.G, across = cg / VEC;
  const int unit = threadIdx.x / p.lanes, l = threadIdx.x % p.lanes;
  const int g = unit % s.G, r = unit / s.G;
  const bool there = r < p.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * p.rows, b0 = static_cast<int64_t>(blockIdx.x) * p.rows;
  const int rounds = static_cast<int>((s.B - b0 + step - 1) / step);                          // of the block
  const int mine = there && b0 + r < s.B ? static_cast<int>((s.B - b0 - r + step - 1) / step) : 0;
  const T* from[SLOTS];
  U* to[SLOTS];
  bool has[SLOTS];
  uint64_t wv[SLOTS][kP], bv[SLOTS][kP];
  using In = Copied<T, VEC>;
  constexpr int kDepth = units_depth(units_bytes(In::kBytes, 0, SLOTS, false));
  extern __shared__ __align__(16) uint8_t smem[];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    const int e = k * p.lanes + l, row = e / across, c = g * cg + e % across * VEC;
    has[k] = there && row < s.N;
    from[k] = x + (b0 + r) * s.x_sample + row * s.x_row + c;
    to[k] = y + ((b0 + r) * s.N + row) * s.C + c;
    channels<VEC>(w, c, has[k], 1.0f, wv[k]);
    channels<VEC>(bias, c, has[k], 0.0f, bv[k]);
  }
  const float n = static_cast<float>(s.N) * static_cast<float>(cg), per = 1.0f / n;
  const int64_t x_step = step * s.x_sample, y_step = step * s.N * s.C;
  float2* stat = stats + (b0 + r) * s.G + g;
  const int64_t stat_step = step * s.G;
  // a thread's places in a stage, and the stages of the sample fetched and of the one worked on
  const uint32_t mine_at = threadIdx.x * In::kBytes, slot_bytes = blockDim.x * In::kBytes, stage_bytes = SLOTS * slot_bytes;
  const uint32_t base = smem_u32(smem) + mine_at;
  uint32_t fetched = 0, used = 0;
  auto fetch = [&](int round) {
    if (round < mine) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (has[k]) In::fetch(base + fetched + k * slot_bytes, from[k]);
    }
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) from[k] += x_step;
    fetched = fetched == (kDepth - 1) * stage_bytes ? 0 : fetched + stage_bytes;
    cp_commit();
  };
#pragma unroll
  for (int round = 0; round < kDepth - 1; ++round) fetch(round);
  for (int round = 0; round < rounds; ++round) {
    uint64_t d[SLOTS][kP], t = 0;
    fetch(round + kDepth - 1);
    cp_wait<kDepth - 1>();
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      Pack<T, VEC> v = Pack<T, VEC>();
      if (In::kCopies) {                           // what was not fetched is replaced, not asked for: nearly all is
        v = In::take(smem, mine_at + used + k * slot_bytes, nullptr);
        if (!(has[k] && round < mine)) v = Pack<T, VEC>();
      } else if (has[k] && round < mine) {         // the pointers are kDepth samples ahead
        v = In::take(smem, 0, from[k] - kDepth * x_step);
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) d[k][i] = v.pair(i);
#pragma unroll
      for (int i = 0; i < kP; ++i) t = f2_add(t, d[k][i]);
    }
    used = used == (kDepth - 1) * stage_bytes ? 0 : used + stage_bytes;
    const float mean = over(lanes_sum(both<VEC>(t), p.lanes), n, per);
    const uint64_t minus = f2_of(-mean);
    t = 0;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      uint64_t u = 0;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        d[k][i] = f2_add(d[k][i], minus);
        u = f2_fma(d[k][i], d[k][i], u);
      }
      if (has[k]) t = f2_add(t, u);
    }
    const float rstd = inverse_sqrt(fmaf(lanes_sum(both<VEC>(t), p.lanes), per, eps));
    if (stats && l == 0 && round < mine) *stat = make_float2(mean, rstd);
    stat += stat_step;
    const uint64_t scale = f2_of(rstd);
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      Pack<U, VEC> o;
#pragma unroll
      for (int i = 0; i < kP; ++i) o.set(i, activate<ACT>(f2_fma(f2_mul(d[k][i], scale), wv[k][i], bv[k][i])));
      if (has[k] && round < mine) *reinterpret_cast<Pack<U, VEC>*>(to[k]) = o;
      to[k] += y_step;
    }
  }
}

enum Mode { kFused, kStats, kApply };

// Tiles: a block's chunk of a slab in registers, the next sample's on its way meanwhile.  parts: (B, chunks, G) pairs of mean
// and summed squared differences between the two kernels of samples that no cluster holds.
template <typename T, typename U, int ACT, int VEC, int MODE>
__global__ void __launch_bounds__(kTileThreads, 3) tiles_kernel(const T* __restrict__ x, U* __restrict__ y, float2* stats,
                                                               const float* __restrict__ w, const float* __restrict__ bias, const Shape s, const Plan p,
                                                               float eps,
                                                               float2* parts) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float part[2][kTileThreads];
  __shared__ float2 mine[kTileThreads];             // a group's mean and squares here
  const int cg = s.C / s.G, across = cg / VEC, groups = p.slab / cg;
  const int v = threadIdx.x % p.V, r = threadIdx.x / p.V, lanes = blockDim.x / p.V, j = v / across;
  // what the statistics' kernel read last is read first
  const int chunk0 = blockIdx.x % p.chunks, slab = blockIdx.x / p.chunks, chunk = MODE == kApply ? p.chunks - 1 - chunk0 : chunk0;
  const int c = slab * p.slab + v * VEC, g = slab * groups + j;
  const int row0 = chunk * p.chunk_rows, rows = min(p.chunk_rows, static_cast<int>(s.N) - row0);
  const bool there = r < lanes && c < s.C, speaks = there && r == 0 && v % across == 0;
  const int n = there && r < rows ? (rows - r + lanes - 1) / lanes : 0;        // this thread's rows
  auto sample = [&](int64_t k) { return MODE == kApply ? s.B - 1 - k : k; };
  const T* from = x + static_cast<int64_t>(row0 + r) * s.x_row + c;
  U* to = y + static_cast<int64_t>(row0 + r) * s.C + c;
  const int64_t x_step = lanes * s.x_row, y_step = static_cast<int64_t>(lanes) * s.C;
  Ahead<T, VEC, kRows> ahead(smem);
  ahead.fetch(from + sample(blockIdx.y) * s.x_sample, x_step, n);
  constexpr int kP = Pack<T, VEC>::kPairs;
  uint64_t wv[kP], bv[kP];
  channels<VEC>(w, c, there, 1.0f, wv);
  channels<VEC>(bias, c, there, 0.0f, bv);
  const float per = 1.0f / (static_cast<float>(s.N) * static_cast<float>(cg));
  const float here = static_cast<float>(rows) * static_cast<float>(cg), per_here = 1.0f / here;
  auto rows_of = [&](int q) { return static_cast<float>(min(p.chunk_rows, static_cast<int>(s.N) - q * p.chunk_rows)); };
  for (int64_t at = blockIdx.y; at < s.B; at += gridDim.y) {
    const int64_t b = sample(at);
    Pack<T, VEC> d[kRows];
    cp_wait_all();
    ahead.take(d);
    float mean, rstd, sum[1] = {0.0f}, sq[1] = {0.0f};
    if constexpr (MODE != kApply) {
      with_rows(n == kRows, [&](auto all) {
        uint64_t t = 0;
#pragma unroll
        for (int k = 0; k < kRows; ++k)
          if (decltype(all)::value || k < n) {
            uint64_t u = d[k].pair(0);
#pragma unroll
            for (int i = 1; i < kP; ++i) u = f2_add(u, d[k].pair(i));
            t = f2_add(t, u);
          }
        sum[0] = both<VEC>(t);
      });
    }
    if (at + gridDim.y < s.B) ahead.fetch(from + sample(at + gridDim.y) * s.x_sample, x_step, n);
    if constexpr (MODE != kApply) {
      group_sums(sum, p.V, lanes, across, v, part[0]);
      mean = over(sum[0], here, per_here);
      with_rows(n == kRows, [&](auto all) {
        uint64_t t = 0;
#pragma unroll
        for (int k = 0; k < kRows; ++k)
          if (decltype(all)::value || k < n) {
            uint64_t u = 0;
#pragma unroll
            for (int i = 0; i < kP; ++i) {
              const uint64_t e = f2_add(d[k].pair(i), f2_of(-mean));
              u = f2_fma(e, e, u);
            }
            t = f2_add(t, u);
          }
        sq[0] = both<VEC>(t);
      });
      group_sums(sq, p.V, lanes, across, v, part[1]);
      if (MODE == kStats) {
        if (speaks) parts[(b * p.chunks + chunk) * s.G + g] = make_float2(mean, sq[0]);
        continue;
      }
      if (p.chunks > 1) {
        // the cluster's blocks have the other chunks
        if (speaks) mine[j] = make_float2(mean, sq[0]);
        cg_::cluster_group cluster = cg_::this_cluster();
        cluster.sync();
        float total = 0.0f;
        for (int q = 0; q < p.chunks; ++q) total = fmaf(cluster.map_shared_rank(mine, q)[j].x, rows_of(q), total);
        mean = total / static_cast<float>(s.N);
        sq[0] = 0.0f;
        for (int q = 0; q < p.chunks; ++q) {
          const float2 theirs = cluster.map_shared_rank(mine, q)[j];
          const float e = theirs.x - mean;
          sq[0] += fmaf(e * e, rows_of(q) * static_cast<float>(cg), theirs.y);
        }
        cluster.sync();                            // every block has read the others' parts
      }
    } else {
      // the chunks' parts, the group's threads in a row taking them in turn: 32 lanes of warp k for group k
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
      __syncthreads();
      for (int k = warp; k < groups && slab * groups + k < s.G; k += warps) {
        const float2* f = parts + b * p.chunks * s.G + slab * groups + k;
        float total = 0.0f;
        for (int q = lane; q < p.chunks; q += 32) total = fmaf(f[static_cast<int64_t>(q) * s.G].x, rows_of(q), total);
#pragma unroll
        for (int m = 16; m; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
        const float m = total / static_cast<float>(s.N);
        float all = 0.0f;
        for (int q = lane; q < p.chunks; q += 32) {
          const float2 t = f[static_cast<int64_t>(q) * s.G];
          const float e = t.x - m;
          all += fmaf(e * e, rows_of(q) * static_cast<float>(cg), t.y);
        }
#pragma unroll
        for (int q = 16; q; q >>= 1) all += __shfl_xor_sync(0xffffffffu, all, q);
        if (lane == 0) mine[k] = make_float2(m, all);
      }
      __syncthreads();
      mean = mine[j].x, sq[0] = mine[j].y;
    }
    if constexpr (MODE != kStats) {
      rstd = inverse_sqrt(fmaf(sq[0], per, eps));
      if (speaks && chunk == 0 && stats) stats[b * s.G + g] = make_float2(mean, rstd);
      U* out = to + b * s.N * s.C;
      uint64_t scale[kP];
#pragma unroll
      for (int i = 0; i < kP; ++i) scale[i] = f2_mul(wv[i], f2_of(rstd));
      with_rows(n == kRows, [&](auto all) {
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          if (decltype(all)::value || k < n) {
            Pack<U, VEC> o;
#pragma unroll
            for (int i = 0; i < kP; ++i) o.set(i, activate<ACT>(f2_fma(f2_add(d[k].pair(i), f2_of(-mean)), scale[i], bv[i])));
            *reinterpret_cast<Pack<U, VEC>*>(out) = o;
          }
          out += y_step;
        }
      });
    }
  }
}

// Wide groups: a block per sample and group, in three passes
template <typename T, typename U, int ACT>
__global__ void __launch_bounds__(256) wide_kernel(const T* __restrict__ x, U* __restrict__ y, float2* stats,
                                                   const float* __restrict__ w, const float* __restrict__ bias, const Shape s,
                                                   float eps) {
  __shared__ double red[8];
  const int cg = s.C / s.G;
  const int64_t n = s.N * cg;
  for (int64_t at = blockIdx.x; at < s.B * s.G; at += gridDim.x) {
    const int64_t b = at / s.G;
    const int c0 = static_cast<int>(at % s.G) * cg;
    const T* xs = x + b * s.x_sample + c0;
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) sum += load_f32(xs + i / cg * s.x_row + i % cg);
    const float mean = block_mean(sum, n, red);
    double sq = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const double d = load_f32(xs + i / cg * s.x_row + i % cg) - mean;
      sq = fma(d, d, sq);
    }
    const float rstd = 1.0f / sqrtf(block_mean(sq, n, red) + eps);
    if (threadIdx.x == 0 && stats) stats[at] = make_float2(mean, rstd);
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const int c = c0 + static_cast<int>(i % cg);
      const int64_t r = i / cg;
      const float xh = (load_f32(x + b * s.x_sample + r * s.x_row + c) - mean) * rstd;
      store_f32(y + (b * s.N + r) * s.C + c, activate1<ACT>(fmaf(w ? w[c] : 1.0f, xh, bias ? bias[c] : 0.0f)));
    }
  }
}

Plan plan_of(const Shape& s, int size, bool aligned) { return make_plan(s, size, num_sms(), aligned, false); }

}  // namespace

size_t forward_workspace(const Shape& s, int size) {
  size_t bytes = 16;
  for (bool aligned : {false, true}) {
    const Plan p = plan_of(s, size, aligned);
    if (p.kind == kTiles && !p.fused) bytes = std::max(bytes, sizeof(float2) * static_cast<size_t>(s.B) * p.chunks * s.G);
  }
  return bytes;
}

namespace {

template <typename T, typename U, int ACT, int VEC>
int run_units(const T* x, U* y, float2* stats, const float* w, const float* bias, const Shape& s, const Plan& p, float eps,
              cudaStream_t st) {
  // rounds are counted in 32 bits: more blocks for more than 2^31 of them (of which the first ones' memory would be full)
  const int64_t blocks = (s.B + p.rows - 1) / p.rows, resident = num_sms() * static_cast<int64_t>(std::max(1, 1024 / p.threads));
  const unsigned grid = static_cast<unsigned>(std::min(blocks, std::max(resident, blocks >> 30)));
  Shape shape = s;
  Plan plan = p;
  void* args[] = {&x, &y, &stats, &w, &bias, &shape, &plan, &eps};
  const void* fn = p.slots == 1   ? reinterpret_cast<const void*>(&units_kernel<T, U, ACT, VEC, 1>)
                   : p.slots == 2 ? reinterpret_cast<const void*>(&units_kernel<T, U, ACT, VEC, 2>)
                                  : reinterpret_cast<const void*>(&units_kernel<T, U, ACT, VEC, 4>);
  return launch_clusters(fn, dim3(grid), dim3(p.threads), units_smem(p, s, sizeof(T), sizeof(U), false), st, args, 1, "group_norm");
}

template <typename T, typename U, int ACT, int VEC>
int run_tiles(const T* x, U* y, float2* stats, const float* w, const float* bias, const Shape& s, const Plan& p, float eps,
              void* ws, cudaStream_t st) {
  const char* what = "group_norm";
  float2* parts = static_cast<float2*>(ws);
  Shape shape = s;
  Plan plan = p;
  void* args[] = {&x, &y, &stats, &w, &bias, &shape, &plan, &eps, &parts};
  const dim3 grid = tiles_grid(s, p, 3, num_sms(), s.B);
  const int smem = Ahead<T, VEC, kRows>::kBytes * kTileThreads;
  if (p.fused)
    return launch_clusters(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kFused>), grid, dim3(p.threads), smem, st, args, p.chunks, what);
  if (int e = launch_clusters(reinterpret_cast<const void*>(&tiles_kernel<T, U, BPC_ACT_NONE, VEC, kStats>), grid, dim3(p.threads), smem, st, args, 1, what))
    return e;
  return launch_clusters(reinterpret_cast<const void*>(&tiles_kernel<T, U, ACT, VEC, kApply>), grid, dim3(p.threads), smem, st, args, 1, what);
}

}  // namespace
}  // namespace gn
}  // namespace bpc

using namespace bpc;
using namespace bpc::gn;

extern "C" int bpc_group_norm_fwd(const void* x, void* y, float* stats, const float* weight, const float* bias,
                                  int64_t B, int64_t N, int32_t C, int32_t G, int64_t x_sample_stride,
                                  int64_t x_row_stride, float eps, int32_t activation, int32_t x_dtype, int32_t y_dtype,
                                  void* workspace, size_t workspace_bytes, bpc_stream_t stream) {
  const Shape s{B, N, C, G, x_sample_stride, x_row_stride, 0, 0};
  const char* what = "group_norm";
  if (int e = check_shape(s, activation, x_dtype, y_dtype, what)) return e;
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(BPC_ERR_ARG, "group_norm: eps must be finite and not negative");
  if (B == 0 || N == 0) return 0;
  if (!x || !y || !workspace) return fail(BPC_ERR_ARG, "group_norm: null buffer");
  const int size = size_of(x_dtype);
  if (!aligned(x, size) || !aligned(y, size_of(y_dtype)) || !aligned(stats, 8) || !aligned(weight, 4) || !aligned(bias, 4) ||
      !aligned(workspace, 16))
    return fail(BPC_ERR_ARG, "group_norm: buffer not aligned to its type (stats: 8 bytes, workspace: 16)");
  if (workspace_bytes < bpc_group_norm_workspace_size(B, N, C, G, x_dtype, 0)) return fail(BPC_ERR_SPACE, "group_norm: workspace too small");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool whole = aligned(x, 16) && aligned(y, 16) && x_sample_stride * size % 16 == 0 && x_row_stride * size % 16 == 0;
  const Plan p = plan_of(s, size, whole);
  return with_types(x_dtype, y_dtype, [&](auto xt, auto yt) {
    return with_act(activation, [&](auto act) {
      typedef typename decltype(xt)::type T;
      typedef typename decltype(yt)::type U;
      constexpr int ACT = decltype(act)::value;
      const T* from = static_cast<const T*>(x);
      U* to = static_cast<U*>(y);
      float2* pairs = reinterpret_cast<float2*>(stats);
      if (p.kind == kWide) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(B * G, 8 * num_sms()));
        wide_kernel<T, U, ACT><<<grid, 256, 0, st>>>(from, to, pairs, weight, bias, s, eps);
        return launched(what);
      }
      if (p.kind == kUnits) {
        if (p.vec == 1) return run_units<T, U, ACT, 1>(from, to, pairs, weight, bias, s, p, eps, st);
        return run_units<T, U, ACT, 16 / sizeof(T)>(from, to, pairs, weight, bias, s, p, eps, st);
      }
      if (p.vec == 1) return run_tiles<T, U, ACT, 1>(from, to, pairs, weight, bias, s, p, eps, workspace, st);
      return run_tiles<T, U, ACT, kTileVec>(from, to, pairs, weight, bias, s, p, eps, workspace, st);
    });
  });
}
