// Token embedding with any number of tokens: the lookup with a scale, and its weight gradient by sorted tokens.
//
//   lookup    y[i, :] = scale W[ids[i], :]                              (a zero row where ids[i] is outside [0, V))
//   gradient  dW[v, :] = scale sum over i with ids[i] = v of gy[i, :]   (ids outside [0, V) contribute nothing)
//
// The products and sums are fp32 and rounded once to the output's type.  The gradient is deterministic.  More than 8 tokens:
// the positions are sorted stably by token (least-significant-digit radix sort), and the sorted rows are summed in that
// order.  Up to 8: every block has a fixed share of the rows, each thread adds its own in order, and the threads' and the
// blocks' sums are added in a fixed order.
#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <utility>

#include <cuda_fp16.h>

#include "bpc.h"
#include "bpc_common.cuh"
#include "bpc_internal.h"
#include "ring_phase.h"

namespace bpc {

namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// VEC elements moved as one access
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// a pack as one access of its whole size
template <int BYTES>
struct Word;
template <> struct Word<16> { typedef uint4 type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };

template <typename P>
__device__ __forceinline__ P load_pack(const void* p) {
  const auto w = *static_cast<const typename Word<sizeof(P)>::type*>(p);
  P x;
  memcpy(&x, &w, sizeof(P));
  return x;
}

template <typename P>
__device__ __forceinline__ void store_pack(void* p, const P& x) {
  typename Word<sizeof(P)>::type w;
  memcpy(&w, &x, sizeof(P));
  *static_cast<typename Word<sizeof(P)>::type*>(p) = w;
}

// ---------------------------------------------------------------------------------------------------------------
// lookup: the threads lie along a row's pieces of VEC channels and several rows, kLookupRows rows per thread in flight
// (one at a time left the stores waiting for the ids' and the table's latency: 110 us at 258,048 rows of 512 fp32 against
// 90, 5.9 TB/s written; bound by HBM).
constexpr int kLookupRows = 4;
constexpr int kLookupBlocks = 4;                          // per SM

// A channel count that no vector width divides: the output as one run of 16-byte stores that cross from row to row (element
// stores took 140 against 92 us at 100,000 rows of 777 fp32).
template <typename I, typename TW, typename TY>
__global__ void __launch_bounds__(256) embed_lookup_flat_kernel(const I* __restrict__ ids, const TW* __restrict__ w,
                                                                TY* __restrict__ y, int64_t total, int V, int C,
                                                                int64_t ldw, float scale) {
  constexpr int K = 16 / sizeof(TY);
  for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u * K < total; u += gridDim.x * 256ll) {
    const int64_t first = u * K;
    int64_t row;
    if (total <= 0xffffffffll) row = static_cast<uint32_t>(first) / static_cast<uint32_t>(C);
    else row = first / C;
    int c = static_cast<int>(first - row * C);
    int64_t id = ids[row];
    Pack<TY, K> o;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (c == C) {
        c = 0;
        ++row;
        id = first + k < total ? static_cast<int64_t>(ids[row]) : -1;
      }
      o.v[k] = from_f32<TY>(id >= 0 && id < V ? scale * to_f32(w[id * ldw + c]) : 0.f);
      ++c;
    }
    if (first + K <= total) {
      store_pack(y + first, o);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (first + k < total) y[first + k] = o.v[k];
    }
  }
}

template <typename I, typename TW, typename TY, int VEC>
__global__ void __launch_bounds__(256, kLookupBlocks) embed_lookup_kernel(const I* __restrict__ ids, const TW* __restrict__ w,
                                                           TY* __restrict__ y, int64_t n, int V, int C, int pieces,
                                                           int rows_at_once, int64_t ldw, float scale) {
  const int tx = threadIdx.x % pieces, ty = threadIdx.x / pieces;
  const int c = (blockIdx.y * pieces + tx) * VEC;
  if (ty >= rows_at_once || c >= C) return;
  const int64_t batch = static_cast<int64_t>(rows_at_once) * kLookupRows;
  for (int64_t r = blockIdx.x * batch + ty; r < n; r += gridDim.x * batch) {
    int64_t id[kLookupRows];
    Pack<TW, VEC> x[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) id[u] = r + u * rows_at_once < n ? static_cast<int64_t>(ids[r + u * rows_at_once]) : -1;
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u)
      if (id[u] >= 0 && id[u] < V) x[u] = load_pack<Pack<TW, VEC>>(w + id[u] * ldw + c);
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      const bool in = id[u] >= 0 && id[u] < V;
      Pack<TY, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f32<TY>(in ? scale * to_f32(x[u].v[e]) : 0.f);
      if (r + u * rows_at_once < n) store_pack(y + (r + u * rows_at_once) * C + c, o);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Stable radix sort of the positions by token into pairs {token, position}, 8 bits a pass.  Positions whose id is outside
// [0, V) get token V: they sort to the end.
constexpr int kDigitBits = 8;
constexpr int kBins = 1 << kDigitBits;

template <typename I>
__device__ __forceinline__ int token_key(I id, int V) {
  return id >= 0 && static_cast<int64_t>(id) < V ? static_cast<int>(id) : V;
}

__device__ __forceinline__ int warp_inclusive(int s, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  return s;
}

// the lanes whose digit is this lane's, from one ballot per bit (a key of none: any lanes)
__device__ __forceinline__ unsigned same_digit(int digit) {
  unsigned same = 0xffffffffu;
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const bool set = digit >> b & 1;
    const unsigned m = __ballot_sync(0xffffffffu, set);
    same &= set ? m : ~m;
  }
  return same;
}

// The ranks of a warp's ROUNDS x 32 consecutive keys among its earlier ones of the same digit; cnt (kBins, the warp's own,
// zero before) counts its digits.  A negative key is none.
template <int ROUNDS, typename N>
__device__ __forceinline__ void warp_ranks(const int (&key)[ROUNDS], int (&rank)[ROUNDS], int shift, N* cnt, int lane) {
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int digit = (key[r] >> shift) & (kBins - 1);
    const unsigned same = same_digit(digit) & __ballot_sync(0xffffffffu, key[r] >= 0);
    const int before = key[r] < 0 ? 0 : cnt[digit];
    rank[r] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (key[r] >= 0 && lane == __ffs(same) - 1) cnt[digit] = static_cast<N>(before + __popc(same));
    __syncwarp();
  }
}

// Up to kClusterKeys positions: one cluster of 8 or 16 CTAs runs every pass in one launch (separate launches of three
// kernels a pass took 66 us for 32,768 positions, most of it latency).  The CTAs exchange digit counts and pairs through
// distributed shared memory: each holds a run of ROUNDS x 1024 places.
constexpr int kClusterThreads = 1024;
constexpr int kClusterKeys = 16 * kClusterThreads * 4;

__device__ __forceinline__ void st_cluster(uint32_t addr, uint16_t v) {
  asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int x, int y) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}

template <typename I, int CTAS, int ROUNDS>
__global__ void __launch_bounds__(kClusterThreads) sort_cluster_kernel(const I* __restrict__ ids, int n, int V, int passes,
                                                                       int2* __restrict__ out) {
  extern __shared__ int2 places[];                         // (ROUNDS x 1024) this CTA's run, and again by this pass's digit
  __shared__ uint16_t cnt[kClusterThreads / 32][kBins];
  __shared__ uint16_t hist[2][CTAS][kBins];                // every CTA's counts of this pass; two, so that a pass may
                                                           // write while a slower CTA still reads the one before
  __shared__ int own_first[kBins], shift_to[kBins];
  __shared__ int warp_sum[2][kBins / 32];
  constexpr int kRun = ROUNDS * kClusterThreads;
  int2* const ordered = places + kRun;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = static_cast<int>(cluster_ctarank());
  const int first = warp * 32 * ROUNDS + lane;             // of this thread's places in the run
  pdl_launch_dependents();
  cluster_arrive_release();                                // every CTA runs before another writes its shared memory
  cluster_wait_acquire();
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * kDigitBits;
    int key[ROUNDS], pos[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int i = cta * kRun + first + r * 32;
      key[r] = -1;
      pos[r] = i;
      if (i < n) {
        if (pass == 0) {
          key[r] = token_key(ids[i], V);
        } else {
          const int2 p = places[first + r * 32];
          key[r] = p.x;
          pos[r] = p.y;
        }
      }
    }
    for (int k = tid; k < kClusterThreads / 32 * kBins / 2; k += kClusterThreads) reinterpret_cast<int*>(cnt)[k] = 0;
    __syncthreads();
    warp_ranks(key, rank, shift, cnt[warp], lane);
    __syncthreads();
    if (tid < kBins) {                                     // this CTA's counts, and each warp's first place among them
      int at = 0;
#pragma unroll 8
      for (int w = 0; w < kClusterThreads / 32; ++w) {
        const int c = cnt[w][tid];
        cnt[w][tid] = static_cast<uint16_t>(at);
        at += c;
      }
      for (int k = 0; k < CTAS; ++k) st_cluster(map_to_cta(smem_u32(&hist[pass & 1][cta][tid]), k), static_cast<uint16_t>(at));
    }
    cluster_arrive_release();                              // counts written, and every run read
    cluster_wait_acquire();
    // each digit's first place in this CTA's own order, and among all the CTAs' pairs
    int total = 0, before = 0, own = 0, s = 0, s_own = 0;
    if (tid < kBins) {
#pragma unroll
      for (int k = 0; k < CTAS; ++k) {
        const int c = hist[pass & 1][k][tid];
        if (k < cta) before += c;
        if (k == cta) own = c;
        total += c;
      }
      s = warp_inclusive(total, lane);
      s_own = warp_inclusive(own, lane);
      if (lane == 31) {
        warp_sum[0][warp] = s;
        warp_sum[1][warp] = s_own;
      }
    }
    __syncthreads();
    if (tid < kBins) {
      int at = s - total + before, at_own = s_own - own;
      for (int w = 0; w < warp; ++w) {
        at += warp_sum[0][w];
        at_own += warp_sum[1][w];
      }
      own_first[tid] = at_own;
      shift_to[tid] = at - at_own;
    }
    __syncthreads();
    // in its own order first, so that the stores to other CTAs run along theirs
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if (key[r] >= 0) {
        const int digit = (key[r] >> shift) & (kBins - 1);
        ordered[own_first[digit] + cnt[warp][digit] + rank[r]] = make_int2(key[r], pos[r]);
      }
    }
    __syncthreads();
    const uint32_t base = smem_u32(places);
    const int here = min(kRun, n - cta * kRun);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int i = tid + r * kClusterThreads;
      if (i < here) {
        const int2 p = ordered[i];
        const int to = i + shift_to[(p.x >> shift) & (kBins - 1)];
        st_cluster(map_to_cta(base + to % kRun * 8, to / kRun), p.x, p.y);
      }
    }
    cluster_arrive_release();                              // the pairs are in their places
    cluster_wait_acquire();
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = tid + r * kClusterThreads;
    if (cta * kRun + i < n) out[cta * kRun + i] = places[i];
  }
}

// More positions: per-tile digit counts, one scan per digit over the tiles, then each tile places its keys.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 8;                            // keys per thread
constexpr int kSortTile = kSortThreads * kSortRounds;

// src: the ids (first pass) or the previous pass's pairs
__device__ __forceinline__ int key_of(const int2* src, int64_t i, int) { return src[i].x; }
template <typename I>
__device__ __forceinline__ int key_of(const I* src, int64_t i, int V) { return token_key(src[i], V); }

template <typename S>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const S* __restrict__ src, int64_t n, int V, int shift,
                                                                  int* __restrict__ counts, int tiles) {
  __shared__ int cnt[kBins];
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) cnt[b] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile + threadIdx.x;
  int key[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int64_t i = base + r * kSortThreads;
    key[r] = i < n ? key_of(src, i, V) : -1;
  }
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int digit = (key[r] >> shift) & (kBins - 1);
    const unsigned same = same_digit(digit) & __ballot_sync(0xffffffffu, key[r] >= 0);
    if (key[r] >= 0 && (threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&cnt[digit], __popc(same));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) counts[static_cast<int64_t>(b) * tiles + blockIdx.x] = cnt[b];
}

// One block per digit: its counts over the tiles become exclusive sums; totals[digit] their sum.
__global__ void __launch_bounds__(256) sort_scan_kernel(int* __restrict__ counts, int* __restrict__ totals, int tiles) {
  __shared__ int warp_sum[8];
  int* row = counts + static_cast<int64_t>(blockIdx.x) * tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + threadIdx.x;
    const int v = t < tiles ? row[t] : 0;
    const int s = warp_inclusive(v, lane);
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    if (t < tiles) row[t] = before + s - v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Places a tile's keys.  Each warp takes a run of kSortRounds x 32 consecutive keys in order, so ranks by (warp, round,
// lane) keep the order of equal digits.
__device__ __forceinline__ int position_of(const int2* src, int64_t i) { return src[i].y; }
template <typename I>
__device__ __forceinline__ int position_of(const I*, int64_t i) { return static_cast<int>(i); }

template <typename S>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const S* __restrict__ src, int64_t n, int V, int shift,
                                                                  const int* __restrict__ offsets,
                                                                  const int* __restrict__ totals, int tiles,
                                                                  int2* __restrict__ out) {
  __shared__ int cnt[kSortWarps][kBins];
  __shared__ int warp_sum[kSortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = threadIdx.x; b < kSortWarps * kBins; b += kSortThreads) (&cnt[0][0])[b] = 0;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * (kSortRounds * 32) + lane;
  int key[kSortRounds], rank[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int64_t i = base + r * 32;
    key[r] = i < n ? key_of(src, i, V) : -1;
  }
  __syncthreads();
  warp_ranks(key, rank, shift, cnt[warp], lane);
  __syncthreads();
  {
    // first place of each digit: the digits below it, then this digit's earlier tiles, then its earlier warps
    static_assert(kBins == kSortThreads, "one thread per digit");
    const int b = threadIdx.x;
    const int v = totals[b];
    const int s = warp_inclusive(v, lane);
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int at = s - v + offsets[static_cast<int64_t>(b) * tiles + blockIdx.x];
    for (int w = 0; w < warp; ++w) at += warp_sum[w];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = cnt[w][b];
      cnt[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    if (key[r] >= 0)
      out[cnt[warp][(key[r] >> shift) & (kBins - 1)] + rank[r]] = make_int2(key[r], position_of(src, base + r * 32));
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The segmented sum.  V row ends and n sorted rows form one path of V + n steps (a row end follows the last row of its
// token), cut into equal runs of `items` steps, one per worker, so that a token with millions of rows and a million
// tokens without any both spread evenly; every row of dW is written once, the empty ones as zeros.  A token whose rows
// cross workers: each worker but the one at its end leaves a partial sum in tail[], the last one its own in head[], and
// wgrad_join_kernel adds them in order.
//   50,021 tokens, 32,768 rows of 1,024 bf16 into fp32: 87 us in all (floor 41), of which the sort 13, the merge about 58 (269
// MB, 4.6 TB/s, mostly the zeros of tokens without a row; 3.7 TB/s of it reach HBM), the join 11.  65,536 rows of 512 over
// 4,096 tokens: sort 17, merge 23, join 20.
struct MergeArgs {
  const int2* pair;    // (n,) {token, row}, sorted by token
  int64_t n, items, workers;
  int V, C, G;         // G lanes per worker
  int64_t ldg;
  float scale;
  void* dw;
  int dw_dtype;
  float* head;         // (workers, C)
  float* tail;
  int2* ends;          // (workers,) {the token of head[] or -1, whether the token of tail[] begins in the worker}
};

// The tokens finished within the first d steps of the path, by the G lanes of a worker together: each step of the search
// probes G places.
__device__ __forceinline__ int64_t path_search(const MergeArgs& a, int64_t d, int G, int l, unsigned mask) {
  int64_t lo = d > a.n ? d - a.n : 0, hi = d < a.V ? d : a.V;            // lo holds: every row consumed
  while (lo < hi) {
    const int64_t step = (hi - lo + G) / (G + 1), at = lo + (l + 1) * step;
    // token at - 1 is finished before step d iff the next row belongs to a later one
    const bool done = at <= hi && (d - at >= a.n || a.pair[d - at].x >= at);
    const int c = __popc(__ballot_sync(mask, done) & mask);
    const int64_t top = lo + (c + 1) * step - 1;
    lo += c * step;
    if (c < G && top < hi) hi = top;                     // below the first probe that failed
  }
  return lo;
}

// Where a worker starts: {tokens finished, rows consumed} after d steps, or, inside a token that ends within `items` rows,
// after that token: the worker before takes the whole of it, so that only the longer tokens are ever cut.
__device__ __forceinline__ int2 path_start(const MergeArgs& a, int64_t d, int G, int l, unsigned mask) {
  const int64_t i = path_search(a, d, G, l, mask), j = d - i;
  if (i < a.V && j > 0 && a.pair[j - 1].x == i) {
    int64_t lo = j, hi = a.n < j + a.items ? a.n : j + a.items;
    if (hi == a.n || a.pair[hi].x != i) {
      while (lo < hi) {                                    // rows up to lo are the token's
        const int64_t step = (hi - lo + G) / (G + 1), at = lo + (l + 1) * step;
        const bool in = at <= hi && a.pair[at - 1].x == i;
        const int c = __popc(__ballot_sync(mask, in) & mask);
        const int64_t top = lo + (c + 1) * step - 1;
        lo += c * step;
        if (c < G && top < hi) hi = top;
      }
      return make_int2(static_cast<int>(i + 1), static_cast<int>(lo));
    }
  }
  return make_int2(static_cast<int>(i), static_cast<int>(j));
}

template <int VEC>
__device__ __forceinline__ void store_row(void* dw, int dtype, int64_t at, const float* acc, float scale) {
  if (dtype == BPC_DTYPE_F32) {
    Pack<float, VEC < 4 ? VEC : 4>* p = reinterpret_cast<Pack<float, VEC < 4 ? VEC : 4>*>(static_cast<float*>(dw) + at);
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      Pack<float, VEC < 4 ? VEC : 4> o;
#pragma unroll
      for (int f = 0; f < (VEC < 4 ? VEC : 4); ++f) o.v[f] = scale * acc[e + f];
      p[e / 4] = o;
    }
  } else if (dtype == BPC_DTYPE_BF16) {
    Pack<__nv_bfloat16, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = __float2bfloat16_rn(scale * acc[e]);
    *reinterpret_cast<Pack<__nv_bfloat16, VEC>*>(static_cast<__nv_bfloat16*>(dw) + at) = o;
  } else {
    Pack<__half, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = __float2half_rn(scale * acc[e]);
    *reinterpret_cast<Pack<__half, VEC>*>(static_cast<__half*>(dw) + at) = o;
  }
}

// rows whose loads are in flight per worker, for the bytes of a lane's pieces
__host__ __device__ constexpr int merge_rows(int bytes) { return bytes >= 32 ? 4 : 8; }

// The asynchronous copy of a piece.  The shortest is 4 bytes: of a 2-byte piece the aligned word around it.
template <int BYTES>
__device__ __forceinline__ void copy_ahead(void* smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(smem)), "l"(global), "n"(BYTES) : "memory");
}

// zeros for a run of memory, by the G lanes of a worker: 16 bytes a lane between its unaligned ends (every type's size is
// a multiple of 2 bytes, and so is the alignment of dW)
__device__ __forceinline__ void zero_run(char* p, int64_t bytes, int l, int G) {
  const int64_t front = (0 - reinterpret_cast<uintptr_t>(p)) & 15, head = front < bytes ? front : bytes;
  for (int64_t b = 2 * l; b < head; b += 2 * G) *reinterpret_cast<uint16_t*>(p + b) = 0;
  const int64_t whole = (bytes - head) / 16;
  uint4* q = reinterpret_cast<uint4*>(p + head);
  for (int64_t k = l; k < whole; k += G) q[k] = make_uint4(0, 0, 0, 0);
  for (int64_t b = head + 16 * whole + 2 * l; b < bytes; b += 2 * G) *reinterpret_cast<uint16_t*>(p + b) = 0;
}

// S pieces of VEC channels per lane, G VEC channels apart (G = 32 lanes where S > 1).  Every lane copies its pieces of the
// rows ahead into its own slots of shared memory (and reads only those, so no barrier is needed): the loads in flight do
// not depend on the registers, which held a block of eight rows to two per SM.  More pieces per lane share a step's
// bookkeeping, which bounded two pieces (88 instructions a step at 50,021 tokens x 1,024).
// FULL: every lane has all S pieces, and dW begins on 16 bytes.
template <typename T, int VEC, int S, bool FULL>
__global__ void __launch_bounds__(256) wgrad_merge_kernel(const T* __restrict__ gy, const __grid_constant__ MergeArgs a) {
  typedef Pack<T, VEC> Piece;
  constexpr int kSlot = sizeof(Piece) < 4 ? 4 : sizeof(Piece);
  constexpr int kRows = merge_rows(S * kSlot);
  extern __shared__ uint4 merge_smem[];                    // slots (kRows, S, 256), then tokens (kRows, 256)
  __shared__ int2 starts[257];
  char* const slots = reinterpret_cast<char*>(merge_smem) + threadIdx.x * kSlot;
  int* const tokens = reinterpret_cast<int*>(reinterpret_cast<char*>(merge_smem) + kRows * S * 256 * kSlot) + threadIdx.x;
  uint32_t odd = 0;                                        // 2-byte pieces: bit u S + q, whether it is its word's upper half
  const int G = S > 1 ? 32 : a.G;
  const int l = threadIdx.x % G, mine = threadIdx.x / G, per_block = 256 / G;
  const int64_t w = blockIdx.x * static_cast<int64_t>(per_block) + mine;
  const int64_t end = a.V + a.n, d0 = min(end, w * a.items), d1 = min(end, d0 + a.items);
  const int shift = (threadIdx.x & 31) / G * G;
  const unsigned mask = (G == 32 ? 0xffffffffu : (1u << G) - 1) << shift;
  pdl_launch_dependents();
  pdl_wait();
  {
    const int2 at = path_start(a, d0, G, l, mask);
    if (l == 0) starts[mine] = at;
    if (mine == per_block - 1) {
      const int2 e = path_start(a, d1, G, l, mask);
      if (l == 0) starts[per_block] = e;
    }
  }
  __syncthreads();
  if (w >= a.workers) return;
  const int i0 = starts[mine].x, i1 = starts[mine + 1].x;
  const int j0 = starts[mine].y, j1 = starts[mine + 1].y;
  // the rows from the loop's place on, and how many are left: a place counted up to 2 kRows beyond the last one would not
  // fit 31 bits where n is 2^31 - 1
  const int2* next = a.pair + j0;
  int left = j1 - j0;
  const int c = (blockIdx.y * S * G + l) * VEC, apart = G * VEC;          // piece q: channels c + q apart ..
  const int pieces = FULL ? S : c < a.C ? min(S, (a.C - c + apart - 1) / apart) : 0;
  bool open = j0 > 0 && i0 < a.V && a.pair[j0 - 1].x == i0;               // token i0 began in an earlier worker
  if (l == 0 && blockIdx.y == 0) a.ends[w] = make_int2(open && i1 > i0 ? i0 : -1, i1 > i0 || !open);
  float acc[S][VEC];
#pragma unroll
  for (int q = 0; q < S; ++q)
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[q][e] = 0.f;
  int tok = i0;
  // ends the tokens up to t: the open one's sum, then the ones without a row
  const auto end_tokens = [&](int t) {
#pragma unroll
    for (int q = 0; q < S; ++q) {
      if (q < pieces) {
        if (open) store_row<VEC>(a.head, BPC_DTYPE_F32, w * a.C + c + q * apart, acc[q], 1.f);
        else store_row<VEC>(a.dw, a.dw_dtype, static_cast<int64_t>(tok) * a.C + c + q * apart, acc[q], a.scale);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[q][e] = 0.f;
    }
    open = false;
    if (FULL && VEC * S >= 4 && a.dw_dtype == BPC_DTYPE_F32) {
      // a warp's pieces of a row are one run of memory: 16 bytes a lane along it, whole sectors in every store
      char* p = reinterpret_cast<char*>(static_cast<float*>(a.dw) + (tok + 1) * static_cast<int64_t>(a.C) +
                                        blockIdx.y * S * 32 * VEC) + l * 16;
      for (int v = tok + 1; v < t; ++v, p += 4ll * a.C)
#pragma unroll
        for (int b = 0; b < VEC * S / 4; ++b) *reinterpret_cast<uint4*>(p + b * 512) = make_uint4(0, 0, 0, 0);
    } else if (blockIdx.y == 0 && tok + 1 < t) {           // whole rows, of every slice
      const int64_t row_bytes = a.C * (a.dw_dtype == BPC_DTYPE_F32 ? 4ll : 2ll);
      zero_run(static_cast<char*>(a.dw) + (tok + 1) * row_bytes, (t - tok - 1) * row_bytes, l, G);
    }
    tok = t;
  };
  // row j from the loop's place on into slot u; the pair of the row after it is read one call ahead
  int2 ahead = left > 0 ? next[0] : make_int2(a.V, 0);
  const char* const lane_gy = reinterpret_cast<const char*>(gy + c);
  const int64_t row_bytes = a.ldg * static_cast<int64_t>(sizeof(T));
  const auto copy_row = [&](int u, int j) {
    if (j < left) {
      const int2 p = ahead;
      if (j + 1 < left) ahead = next[j + 1];
      tokens[u * 256] = p.x;
      if (p.x < a.V) {                                     // V: a position without a token
        const char* row = lane_gy + p.y * row_bytes;
#pragma unroll
        for (int q = 0; q < S; ++q)
          if (q < pieces) {
            if constexpr (sizeof(Piece) >= 4) {
              copy_ahead<kSlot>(slots + (u * S + q) * 256 * kSlot, row + q * apart * sizeof(T));
            } else {
              const uintptr_t at = reinterpret_cast<uintptr_t>(row + q * apart * sizeof(T));
              const uint32_t bit = 1u << (u * S + q);
              odd = at & 2 ? odd | bit : odd & ~bit;
              copy_ahead<4>(slots + (u * S + q) * 256 * kSlot, reinterpret_cast<const void*>(at & ~static_cast<uintptr_t>(3)));
            }
          }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int u = 0; u < kRows - 1; ++u) copy_row(u, u);
  bool more = true;
  for (; more && left > 0; left -= kRows, next += kRows) {
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (!more || u >= left) break;
      copy_row((u + kRows - 1) % kRows, u + kRows - 1);   // into the slot that the step before read
      asm volatile("cp.async.wait_group %0;" ::"n"(kRows - 1) : "memory");
      const int t = tokens[u * 256];
      if (t >= a.V) {                                      // the ones without a token are the last
        more = false;
        break;
      }
      if (tok < t) end_tokens(t);
#pragma unroll
      for (int q = 0; q < S; ++q) {
        if (q < pieces) {
          const Piece x = load_pack<Piece>(slots + (u * S + q) * 256 * kSlot + (sizeof(Piece) < 4 ? odd >> (u * S + q) << 1 & 2 : 0));
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[q][e] += to_f32(x.v[e]);
        }
      }
    }
  }
  if (tok < i1) end_tokens(i1);
  if (i1 < a.V && j1 > 0 && a.pair[j1 - 1].x == i1) {
#pragma unroll
    for (int q = 0; q < S; ++q)
      if (q < pieces) store_row<VEC>(a.tail, BPC_DTYPE_F32, w * a.C + c + q * apart, acc[q], 1.f);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A warp per token that crosses workers and kJoinChannels channels: the tails of the workers since its first row, then the last
// one's head, in fp64.  One with more than kLongJoin tails is left to the block's warps together, each a fixed share.
constexpr int kLongJoin = 64;
constexpr int kJoinWarps = 8;
constexpr int kJoinRun = 4;
constexpr int kJoinChannels = 128;

template <int VEC>
__global__ void __launch_bounds__(kJoinWarps * 32, 3) wgrad_join_kernel(const __grid_constant__ MergeArgs a) {
  __shared__ double red[kJoinWarps][32 * VEC];
  __shared__ int64_t task_worker[kJoinWarps][kJoinRun], task_first[kJoinWarps][kJoinRun], task_token[kJoinWarps][kJoinRun];
  __shared__ int tasks[kJoinWarps];
  typedef Pack<float, VEC> Piece;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c_from = blockIdx.y * kJoinChannels, c_to = min(a.C, c_from + kJoinChannels);
  pdl_wait();
  // s += tails v0, v0 + by .. below v1, at this lane's channels
  const auto add_tails = [&](double (&s)[VEC], int64_t v0, int64_t v1, int by, int c) {
    for (int64_t v = v0; v < v1; v += 8 * by) {
      Piece x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (v + u * by < v1) x[u] = load_pack<Piece>(a.tail + (v + u * by) * a.C + c);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (v + u * by < v1)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[e] += x[u].v[e];
    }
  };
  const auto finish = [&](const double (&s)[VEC], int64_t w, int64_t t, int c) {
    const Piece h = load_pack<Piece>(a.head + w * a.C + c);
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = static_cast<float>(s[e] + h.v[e]);
    store_row<VEC>(a.dw, a.dw_dtype, t * a.C + c, f, a.scale);
  };
  // a warp looks at kJoinRun workers at once; few of them end a token that was cut
  const int64_t runs = (a.workers + kJoinRun - 1) / kJoinRun;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kJoinWarps; base < runs;
       base += static_cast<int64_t>(gridDim.x) * kJoinWarps) {
    const int64_t mine = (base + warp) * kJoinRun + lane;
    const int token = lane < kJoinRun && mine < a.workers ? a.ends[mine].x : -1;
    unsigned cut = __ballot_sync(0xffffffffu, token >= 0);
    int longs = 0;
    while (cut) {
      const int at_lane = __ffs(cut) - 1;
      cut &= cut - 1;
      const int64_t w = (base + warp) * kJoinRun + at_lane, t = __shfl_sync(0xffffffffu, token, at_lane);
      // the nearest worker before w whose tail's token begins in it, 128 at a time: the first of token t
      int64_t first = 0;
      for (int64_t top = w - 1; top >= 0; top -= 128) {
        unsigned begins[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t v = top - 32 * u - lane;
          begins[u] = __ballot_sync(0xffffffffu, v < 0 || a.ends[v].y);
        }
        int at = 128;
#pragma unroll
        for (int u = 3; u >= 0; --u)
          if (begins[u]) at = 32 * u + __ffs(begins[u]) - 1;
        if (at < 128) {
          first = top - at;
          break;
        }
      }
      if (w - first <= kLongJoin) {
        for (int c = c_from + lane * VEC; c < c_to; c += 32 * VEC) {
          double s[VEC] = {};
          add_tails(s, first, w, 1, c);
          finish(s, w, t, c);
        }
      } else {
        if (lane == 0) {
          task_worker[warp][longs] = w;
          task_first[warp][longs] = first;
          task_token[warp][longs] = t;
        }
        ++longs;
      }
    }
    if (lane == 0) tasks[warp] = longs;
    if (!__syncthreads_or(longs)) continue;
    for (int k = 0; k < kJoinWarps * kJoinRun; ++k) {
      const int from = k / kJoinRun, task = k % kJoinRun;
      if (task >= tasks[from]) continue;
      const int64_t v1 = task_worker[from][task], v0 = task_first[from][task], t = task_token[from][task];
      for (int c0 = c_from; c0 < c_to; c0 += 32 * VEC) {
        const int c = c0 + lane * VEC;
        double s[VEC] = {};
        if (c < c_to) add_tails(s, v0 + warp, v1, kJoinWarps, c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) red[warp][lane * VEC + e] = s[e];
        __syncthreads();
        if (warp == 0 && c < c_to) {
          for (int q = 1; q < kJoinWarps; ++q)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[e] += red[q][lane * VEC + e];
          finish(s, v1, t, c);
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Few tokens (V <= kFewTokens; the detector tokens of this library's networks are 4 or 5): no sort.  The rows are read
// once in their own order.  A ninth warp copies them ahead into a ring of shared memory (bulk copies: the bytes in
// flight depend neither on registers nor on the load units).  The threads of the other eight lie along a row's pieces
// of VEC channels and several rows; each keeps one sum per token in registers and adds its piece under one predicate per
// token.  A block adds its threads' sums in order, wgrad_few_join_kernel the blocks' in fp64.
//   Bound by HBM: 10.8 M rows of 96 bf16 and four tokens take 354 us, 6.0 TB/s (0.91 of a measured copy; 324 us on
// another B200), with the issue slots 0.72 busy (4 tokens: some 70 instructions per 512 bytes).  Tried and slower at that size: sorting (2,144 us), sums in
// shared memory indexed by token (609), cp.async rings per thread (427, bound by the load unit), rows listed by token by
// the ninth warp (427) or by ballots of the adding warps (444).  Eight is the most tokens: groups of eight that read the
// rows again from L2 took 176 us against 127 sorted (20 tokens, 1 M rows of 64 bf16).
constexpr int kFewTokens = 8;
constexpr int kFewThreads = 256;                          // that add
constexpr int kFewStages = 4;                             // of 64 bytes per adding thread: 64 KB
constexpr int kFewBlocksPerSm = 3;
constexpr uint64_t kFewTimeoutNs = 2000000000ull;         // bound of every wait

enum FewMode : int {
  kFewWhole = 0,       // a stage's rows are one run of memory: one bulk copy
  kFewRows = 1,        // one per row (16-byte pieces at a row stride, or a slice of the channels)
  kFewDirect = 2,      // not aligned for bulk copies: the rows are read from global memory
};

struct FewPlan {
  int vec, mode;
  int pieces;          // of vec channels per row and slice
  int rows_at_once;    // kFewThreads / pieces
  int slices;          // of the channels (gridDim.y)
  int batch;           // rows of a stage
  uint32_t pitch;      // bytes from row to row in shared memory
  int64_t blocks, rows_per_block;
};

struct FewArgs {
  FewPlan p;
  const void* gy;
  const void* ids;
  int id_bytes;
  int64_t n, ldg;
  int V, C;
  float scale;
  void* dw;
  int dw_dtype;
  float* partial;      // (gridDim.x, V, C), unused when one block covers the rows
  int* status;         // watchdog word of the op entry points
};

__device__ __forceinline__ int small_token(const int32_t* p) { return __ldg(p); }
__device__ __forceinline__ int small_token(const int64_t* p) {
  const int2 w = __ldg(reinterpret_cast<const int2*>(p));
  return w.y == 0 ? w.x : -1;                              // an id that does not fit 32 bits is none
}

template <int VEC>
__device__ __forceinline__ void add_if(float (&s)[VEC], const float (&x)[VEC], int t, int v) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = t == v ? s[e] + x[e] : s[e];
}

template <typename T, typename I, int VEC, int NV>
__global__ void __launch_bounds__(kFewThreads + 32) wgrad_few_kernel(const __grid_constant__ FewArgs a) {
  extern __shared__ uint4 few_smem_base[];
  __shared__ __align__(8) uint64_t full[kFewStages], empty[kFewStages];
  __shared__ int abort;
  typedef Pack<T, VEC> Piece;
  constexpr int kRows = 64 / sizeof(Piece);                // rows per thread and stage
  constexpr int kAhead = 4;                                // rows whose tokens are read ahead
  const FewPlan& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = blockIdx.x * p.rows_per_block;
  const int rows = static_cast<int>(min(a.n - r0, p.rows_per_block));
  const int c0 = blockIdx.y * p.pieces * VEC;
  const int width = min(p.pieces * VEC, a.C - c0);         // channels of this slice
  const T* gp = static_cast<const T*>(a.gy) + r0 * a.ldg + c0;
  const int TY = p.rows_at_once, batch = kRows * TY;
  const int copied = p.mode == kFewDirect ? 0 : rows / batch;          // the stages that pass through the ring
  volatile int* gave_up = &abort;
  if (tid == 0) {
    abort = 0;
    for (int k = 0; k < kFewStages; ++k) {
      mbar_init(smem_u32(&full[k]), 1);
      mbar_init(smem_u32(&empty[k]), kFewThreads / 32);
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == kFewThreads / 32) {
    const uint32_t ring = smem_u32(few_smem_base), row_bytes = width * sizeof(T);
    int issued = 0;
    for (int k = 0; k < copied; ++k) {
      const int q = k % kFewStages;
      // the warp leaves as a whole: a lane that gave up alone would leave the others at the barriers below
      if (k >= kFewStages &&
          !__all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[q]), ring_parity(k - kFewStages, kFewStages), gave_up,
                                             a.status, kFewTimeoutNs)))
        break;
      __syncwarp();
      const uint32_t dst = ring + q * batch * p.pitch, bar = smem_u32(&full[q]);
      const T* src = gp + static_cast<int64_t>(k) * batch * a.ldg;
      if (lane == 0) mbar_arrive_expect_tx(bar, batch * row_bytes);
      __syncwarp();
      if (p.mode == kFewWhole) {
        if (lane == 0) bulk_load(dst, src, batch * row_bytes, bar);
      } else {
        for (int r = lane; r < batch; r += 32) bulk_load(dst + r * p.pitch, src + r * a.ldg, row_bytes, bar);
      }
      issued = k + 1;
    }
    __syncthreads();
    // after a wait that ran out: copies under way still write this block's memory, give them as long again
    if (abort && lane == 0) {
      volatile int never = 0;
      for (int q = 0; q < kFewStages && q < issued; ++q)
        mbar_wait(smem_u32(&full[q]), ring_parity(ring_last_use(issued, q, kFewStages), kFewStages), &never, nullptr,
                  kFewTimeoutNs);
    }
    __syncthreads();
    return;
  }

  float s[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[v][e] = 0.f;
  const int x = tid % p.pieces, y = tid / p.pieces;
  const bool on = y < TY && x * VEC < width;
  const auto add = [&](const Piece piece, int t) {         // a token of V or more meets no sum that is read
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = to_f32(piece.v[e]);
#pragma unroll
    for (int v = 0; v < NV; ++v) add_if(s[v], f, t, v);
  };
  const I* idp = static_cast<const I*>(a.ids) + r0 + (on ? y : 0);
  int next[kAhead];                                        // the tokens of this thread's next rows
  const auto tokens = [&](int r) {                         // rows r, r + TY .. of this thread's stages: all in range
#pragma unroll
    for (int u = 0; u < kAhead; ++u) next[u] = small_token(idp + (r + u * TY));
  };
  const char* const mine = reinterpret_cast<const char*>(few_smem_base) + y * p.pitch + x * sizeof(Piece);
  const uint32_t row_step = TY * p.pitch, stage_step = batch * p.pitch;
  if (copied) tokens(0);
  uint32_t q = 0, parity = 0;
  for (int k = 0; k < copied; ++k) {
    const bool ok = mbar_wait(smem_u32(&full[q]), parity, gave_up, a.status, kFewTimeoutNs);
    const char* at = mine + q * stage_step;
#pragma unroll
    for (int j = 0; j < kRows; j += kAhead) {
      int t[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) t[u] = next[u];
      if (j + kAhead < kRows || k + 1 < copied) tokens((j + kAhead) * TY);
      if (on) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) add(load_pack<Piece>(at + (j + u) * row_step), t[u]);
      }
    }
    idp += batch;
    if (!__all_sync(0xffffffffu, ok)) break;               // as a warp: see above
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&empty[q]));
    if (++q == kFewStages) {
      q = 0;
      parity ^= 1;
    }
  }
  if (on) {                                                // what does not fill a stage
    for (int r = copied * batch + y; r < rows; r += TY)
      add(load_pack<Piece>(gp + static_cast<int64_t>(r) * a.ldg + x * VEC),
          small_token(static_cast<const I*>(a.ids) + r0 + r));
  }
  __syncthreads();                                         // the ring is read: its memory takes the sums
  __syncthreads();
  float* sums = reinterpret_cast<float*>(few_smem_base);   // (V, VEC, kFewThreads)
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v < a.V)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sums[(v * VEC + e) * kFewThreads + tid] = s[v][e];
  pdl_launch_dependents();
  asm volatile("bar.sync 1, %0;" ::"n"(kFewThreads) : "memory");            // the eight warps that add
  for (int i = tid; i < a.V * p.pieces; i += kFewThreads) {
    const int v = i / p.pieces, xx = i - v * p.pieces;
    if (xx * VEC >= width) continue;
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float* q = sums + (v * VEC + e) * kFewThreads + xx;
      o[e] = 0.f;
      for (int yy = 0; yy < p.rows_at_once; ++yy) o[e] += q[yy * p.pieces];
    }
    const int cc = c0 + xx * VEC;
    if (gridDim.x == 1) {
      store_row<VEC>(a.dw, a.dw_dtype, static_cast<int64_t>(v) * a.C + cc, o, a.scale);
    } else {
      float* out = a.partial + (static_cast<int64_t>(blockIdx.x) * a.V + v) * a.C + cc;
#pragma unroll
      for (int e = 0; e < VEC; ++e) out[e] = o[e];
    }
  }
}

// 32 sums a block, its warps each a fixed share of the blocks' partial sums, in fp64
__global__ void __launch_bounds__(1024) wgrad_few_join_kernel(const float* __restrict__ partial, int blocks, int n,
                                                              float scale, void* dw, int dw_dtype) {
  __shared__ double red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  const int i = blockIdx.x * 32 + lane;
  double s = 0.0;
  if (i < n) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += 32) s += partial[static_cast<int64_t>(b) * n + i];
  }
  red[warp][lane] = s;
  __syncthreads();
  // transposed: warp w now holds the 32 shares of sum w
  s = red[lane][warp];
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  const int o = blockIdx.x * 32 + warp;
  if (lane == 0 && o < n) {
    const float f = static_cast<float>(s);
    store_row<1>(dw, dw_dtype, o, &f, scale);
  }
}

int dtype_size(int32_t dtype) { return dtype == BPC_DTYPE_F32 ? 4 : dtype == BPC_DTYPE_BF16 || dtype == BPC_DTYPE_F16 ? 2 : 0; }

// Workspace layout of the gradient by sorted tokens
struct WgradPlan {
  int passes, tiles, G;
  int64_t items, workers;
  size_t pair[2], counts, totals, head, tail, ends, bytes;
};

// The most blocks along the rows; few_plan's slices are the fewest with eight channels a piece.  Three blocks per SM is what
// fits of the variants of up to 4 tokens (72 registers at most).  Of eight 16-bit channels a piece two fit at 5 tokens (79)
// and at 6 to 8 (112), one of bf16 with int64 ids there (113): the grid is then one and a half waves, or three.
int64_t few_most(int slices) { return std::max<int64_t>(1, kFewBlocksPerSm * static_cast<int64_t>(num_sms()) / slices); }

// Few tokens: how a block reads its rows, by alignment and row length.
FewPlan few_plan(const void* gy, const void* dw, int64_t n, int C, int64_t ldg, int size) {
  FewPlan p;
  const auto fits = [&](int vec) {
    return C % vec == 0 && ldg % vec == 0 && reinterpret_cast<uintptr_t>(gy) % (vec * size) == 0 &&
           reinterpret_cast<uintptr_t>(dw) % 16 == 0;
  };
  p.vec = 16 / size;
  while (p.vec > 1 && !fits(p.vec)) p.vec /= 2;
  const int units = (C + p.vec - 1) / p.vec;
  p.slices = (units + kFewThreads - 1) / kFewThreads;
  p.pieces = (units + p.slices - 1) / p.slices;
  p.rows_at_once = kFewThreads / p.pieces;
  p.pitch = static_cast<uint32_t>(p.pieces) * p.vec * size;
  // 64 bytes per thread and stage: narrower pieces take more rows, so that every whole stage begins on 16 bytes
  p.batch = p.rows_at_once * (64 / (p.vec * size));
  if (reinterpret_cast<uintptr_t>(gy) % 16) p.mode = kFewDirect;
  else if (ldg == C && p.slices == 1) p.mode = kFewWhole;
  else if (p.vec * size == 16) p.mode = kFewRows;
  else p.mode = kFewDirect;
  // a whole number of stages per block, unless there are too few rows to fill the GPU that way; at least 8 rows, and a
  // multiple of 8, which begins on 16 bytes too
  const int64_t most = few_most(p.slices);
  int64_t per = (n + most - 1) / most;
  if (per >= 2 * p.batch) per = (per + p.batch - 1) / p.batch * p.batch;
  p.rows_per_block = (per + 7) / 8 * 8;
  p.blocks = (n + p.rows_per_block - 1) / p.rows_per_block;
  return p;
}

// the ring, or the block's sums after it
int few_smem(const FewPlan& p, int V) {
  const int ring = p.mode == kFewDirect ? 0 : static_cast<int>(kFewStages * p.batch * p.pitch);
  return std::max(ring, V * kFewThreads * 4 * p.vec);
}

size_t few_bytes(int64_t n, int32_t V, int32_t C) {
  const int slices = ((C + 7) / 8 + kFewThreads - 1) / kFewThreads;
  return sizeof(float) * V * C * static_cast<size_t>(std::min((n + 7) / 8, few_most(slices)));
}

WgradPlan wgrad_plan(int64_t n, int32_t V, int32_t C) {
  WgradPlan p;
  int bits = 1;
  while (bits < 32 && (static_cast<int64_t>(1) << bits) <= V) ++bits;      // tokens are in [0, V]
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.tiles = static_cast<int>((n + kSortTile - 1) / kSortTile);
  p.G = 1;
  while (p.G < 32 && p.G * 4 < C) p.G *= 2;
  // about 32 warps per SM over the workers and the slices of 512 channels, at least 8 steps a worker (a step is some
  // hundred instructions of one warp in a row: 12 longer workers' warps per SM took half as long again).  16 steps at least
  // take longer where the rows spread over the tokens (3,000 rows of 333 over 50 tokens: 21.8 us of GPU time against 16.0)
  // and 8 where half of them are one token's, whose parts one block joins (200,000 rows of 8 over 300 tokens: 350 against 200)
  const int64_t target = std::max<int64_t>(1, static_cast<int64_t>(num_sms()) * 32 * (32 / p.G) / ((C + 511) / 512));
  p.items = std::max<int64_t>(8, (V + n + target - 1) / target);
  p.workers = (V + n + p.items - 1) / p.items;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 255) & ~static_cast<size_t>(255);
    return r;
  };
  for (int k = 0; k < 2; ++k) p.pair[k] = take(sizeof(int2) * n);
  p.counts = take(sizeof(int) * kBins * static_cast<size_t>(p.tiles));
  p.totals = take(sizeof(int) * kBins);
  p.head = take(sizeof(float) * p.workers * C);
  p.tail = take(sizeof(float) * p.workers * C);
  p.ends = take(sizeof(int2) * p.workers);
  p.bytes = at;
  return p;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

template <typename I, typename TW, typename TY>
int lookup_launch(const void* ids, const void* w, void* y, int64_t n, int V, int C, int64_t ldw, float scale,
                  cudaStream_t s) {
  constexpr int kVec = 16 / (sizeof(TW) > sizeof(TY) ? sizeof(TW) : sizeof(TY));
  const bool wide = C % kVec == 0 && ldw % kVec == 0 && reinterpret_cast<uintptr_t>(w) % (kVec * sizeof(TW)) == 0 &&
                    reinterpret_cast<uintptr_t>(y) % (kVec * sizeof(TY)) == 0;
  if (!wide && C > 1 && reinterpret_cast<uintptr_t>(y) % 16 == 0) {
    const int64_t stores = (n * C * static_cast<int64_t>(sizeof(TY)) + 15) / 16;
    const int grid = static_cast<int>(std::min<int64_t>((stores + 255) / 256, static_cast<int64_t>(num_sms()) * 8));
    embed_lookup_flat_kernel<I, TW, TY><<<grid, 256, 0, s>>>(static_cast<const I*>(ids), static_cast<const TW*>(w),
                                                             static_cast<TY*>(y), n * C, V, C, ldw, scale);
    return launched("embed_lookup_flat_kernel");
  }
  const int units = wide ? C / kVec : C;
  const int slices = (units + 255) / 256, pieces = (units + slices - 1) / slices, rows_at_once = 256 / pieces;
  const int64_t blocks = (n + rows_at_once * kLookupRows - 1) / (rows_at_once * kLookupRows);
  // one wave of blocks with equal shares of the rows
  const int64_t rounds = (blocks + num_sms() * kLookupBlocks - 1) / (num_sms() * kLookupBlocks);
  const dim3 grid(static_cast<unsigned>((blocks + rounds - 1) / rounds), slices);
  const auto run = [&](auto kernel) {
    kernel<<<grid, 256, 0, s>>>(static_cast<const I*>(ids), static_cast<const TW*>(w), static_cast<TY*>(y), n, V, C, pieces,
                                rows_at_once, ldw, scale);
  };
  if (wide) run(embed_lookup_kernel<I, TW, TY, kVec>);
  else run(embed_lookup_kernel<I, TW, TY, 1>);
  return launched("embed_lookup_kernel");
}

template <typename I, typename TW>
int lookup_by_y(const void* ids, const void* w, void* y, int64_t n, int V, int C, int64_t ldw, float scale,
                int32_t y_dtype, cudaStream_t s) {
  if (y_dtype == BPC_DTYPE_F32) return lookup_launch<I, TW, float>(ids, w, y, n, V, C, ldw, scale, s);
  if (y_dtype == BPC_DTYPE_BF16) return lookup_launch<I, TW, __nv_bfloat16>(ids, w, y, n, V, C, ldw, scale, s);
  return lookup_launch<I, TW, __half>(ids, w, y, n, V, C, ldw, scale, s);
}

template <typename I>
int lookup_by_w(const void* ids, const void* w, void* y, int64_t n, int V, int C, int64_t ldw, float scale,
                int32_t w_dtype, int32_t y_dtype, cudaStream_t s) {
  if (w_dtype == BPC_DTYPE_F32) return lookup_by_y<I, float>(ids, w, y, n, V, C, ldw, scale, y_dtype, s);
  if (w_dtype == BPC_DTYPE_BF16) return lookup_by_y<I, __nv_bfloat16>(ids, w, y, n, V, C, ldw, scale, y_dtype, s);
  return lookup_by_y<I, __half>(ids, w, y, n, V, C, ldw, scale, y_dtype, s);
}

template <typename S>
int sort_pass(const S* src, int64_t n, int V, int shift, int tiles, int* counts, int* totals, int2* out, cudaStream_t s) {
  sort_count_kernel<S><<<tiles, kSortThreads, 0, s>>>(src, n, V, shift, counts, tiles);
  if (int e = launched("sort_count_kernel")) return e;
  sort_scan_kernel<<<kBins, 256, 0, s>>>(counts, totals, tiles);
  if (int e = launched("sort_scan_kernel")) return e;
  sort_place_kernel<S><<<tiles, kSortThreads, 0, s>>>(src, n, V, shift, counts, totals, tiles, out);
  return launched("sort_place_kernel");
}

// Whether the kernel's cluster can be resident on the current device (a partition of a GPU may have no room for 16 CTAs);
// asked once per device and kernel.
bool cluster_fits(const void* fn, const cudaLaunchConfig_t& lc) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, bool> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lk(mu);
  const auto it = known.find({dev, fn});
  if (it != known.end()) return it->second;
  int clusters = 0;
  cudaError_t e = cudaSuccess;
  if (lc.gridDim.x > 8) e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, fn, &lc);
  if (e != cudaSuccess) cudaGetLastError();
  return known[{dev, fn}] = e == cudaSuccess && clusters > 0;
}

// *launched: whether the cluster can be resident here and was launched
template <typename I, int CTAS, int ROUNDS>
int sort_cluster_rounds(const I* ids, int n, int V, int passes, int2* out, bool* launched, cudaStream_t s) {
  const auto fn = sort_cluster_kernel<I, CTAS, ROUNDS>;
  const int smem = 2 * ROUNDS * kClusterThreads * static_cast<int>(sizeof(int2));
  if (int e = allow_smem(reinterpret_cast<const void*>(fn), smem)) return e;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(CTAS);
  lc.blockDim = dim3(kClusterThreads);
  lc.dynamicSmemBytes = smem;
  lc.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CTAS;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  *launched = cluster_fits(reinterpret_cast<const void*>(fn), lc);
  if (!*launched) return 0;
  const cudaError_t e = cudaLaunchKernelEx(&lc, fn, ids, n, V, passes, out);
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string("sort_cluster_kernel launch: ") + cudaGetErrorString(e));
}

template <typename I>
int sort_cluster(const I* ids, int n, int V, int passes, int2* out, bool* launched, cudaStream_t s) {
  if (n <= 8 * kClusterThreads) return sort_cluster_rounds<I, 8, 1>(ids, n, V, passes, out, launched, s);
  if (n <= 16 * kClusterThreads) return sort_cluster_rounds<I, 16, 1>(ids, n, V, passes, out, launched, s);
  if (n <= 32 * kClusterThreads) return sort_cluster_rounds<I, 16, 2>(ids, n, V, passes, out, launched, s);
  return sort_cluster_rounds<I, 16, 4>(ids, n, V, passes, out, launched, s);
}

// *sorted: where the pairs are.  BPC_EMBED_SORT=passes selects the launches per pass for every size (the same pairs).
template <typename I>
int sort_ids(const I* ids, int64_t n, int V, const WgradPlan& p, int2* const (&pair)[2], int* counts, int* totals,
             const int2** sorted, cudaStream_t s) {
  *sorted = pair[0];
  const char* how = std::getenv("BPC_EMBED_SORT");
  if (n <= kClusterKeys && !(how && std::strcmp(how, "passes") == 0)) {
    bool launched = false;
    const int e = sort_cluster(ids, static_cast<int>(n), V, p.passes, pair[0], &launched, s);
    if (e || launched) return e;
  }
  if (int e = sort_pass(ids, n, V, 0, p.tiles, counts, totals, pair[0], s)) return e;
  for (int k = 1; k < p.passes; ++k) {
    if (int e = sort_pass(*sorted, n, V, k * kDigitBits, p.tiles, counts, totals, pair[k & 1], s)) return e;
    *sorted = pair[k & 1];
  }
  return 0;
}

template <typename T, int VEC, int S, bool FULL>
int merge_launch_pieces(const T* gy, MergeArgs a, cudaStream_t s) {
  if (S > 1) a.G = 32;
  while (S == 1 && a.G > 1 && a.G / 2 * VEC >= a.C) a.G /= 2;              // no more lanes than pieces
  const int64_t blocks = (a.workers + 256 / a.G - 1) / (256 / a.G);
  const dim3 grid(static_cast<unsigned>(blocks), (a.C + a.G * VEC * S - 1) / (a.G * VEC * S));
  void* args[] = {&gy, &a};
  const void* fn = reinterpret_cast<const void*>(&wgrad_merge_kernel<T, VEC, S, FULL>);
  constexpr int kSlots = S * std::max(4, VEC * static_cast<int>(sizeof(T)));
  constexpr int kSmem = merge_rows(kSlots) * 256 * (kSlots + static_cast<int>(sizeof(int)));
  if (int e = allow_smem(fn, kSmem)) return e;
  if (int e = launch_pdl(fn, grid, dim3(256), kSmem, s, args, 1, "wgrad_merge_kernel")) return e;
  void* join_args[] = {&a};
  const int64_t join = std::min<int64_t>((a.workers + kJoinWarps * kJoinRun - 1) / (kJoinWarps * kJoinRun), 8 * num_sms());
  return launch_pdl(reinterpret_cast<const void*>(&wgrad_join_kernel<(VEC < 4 ? VEC : 4)>),
                    dim3(static_cast<unsigned>(join), (a.C + kJoinChannels - 1) / kJoinChannels),
                    dim3(kJoinWarps * 32), 0, s, join_args, 1, "wgrad_join_kernel");
}

template <typename T, int VEC, int S>
int merge_launch_full(const T* gy, const MergeArgs& a, cudaStream_t s) {
  if (S > 1 && a.C % (32 * VEC * S) == 0 && reinterpret_cast<uintptr_t>(a.dw) % 16 == 0)
    return merge_launch_pieces<T, VEC, S, true>(gy, a, s);
  return merge_launch_pieces<T, VEC, S, false>(gy, a, s);
}

template <typename T, int VEC>
int merge_launch_vec(const T* gy, const MergeArgs& a, cudaStream_t s) {
  if constexpr (VEC < 8) {                                 // at most 512 channels per worker
    if (a.C > 64 * VEC) return merge_launch_full<T, VEC, 4>(gy, a, s);
  }
  return a.C > 32 * VEC ? merge_launch_full<T, VEC, 2>(gy, a, s) : merge_launch_full<T, VEC, 1>(gy, a, s);
}

template <typename T>
int merge_launch(const void* gy, const MergeArgs& a, cudaStream_t s) {
  const auto fits = [&](int vec) {
    return a.C % vec == 0 && a.ldg % vec == 0 && reinterpret_cast<uintptr_t>(gy) % (vec * sizeof(T)) == 0 &&
           reinterpret_cast<uintptr_t>(a.dw) % std::min(16, vec * dtype_size(a.dw_dtype)) == 0;
  };
  const T* g = static_cast<const T*>(gy);
  if constexpr (sizeof(T) == 2) {
    if (fits(8)) return merge_launch_vec<T, 8>(g, a, s);
  }
  if (fits(4)) return merge_launch_vec<T, 4>(g, a, s);
  if (fits(2)) return merge_launch_vec<T, 2>(g, a, s);
  return merge_launch_vec<T, 1>(g, a, s);
}

template <typename T, typename I, int VEC, int NV>
int few_launch_tokens(const FewArgs& a, cudaStream_t s) {
  const auto fn = wgrad_few_kernel<T, I, VEC, NV>;
  const int smem = few_smem(a.p, a.V);
  if (int e = allow_smem(reinterpret_cast<const void*>(fn), smem)) return e;
  fn<<<dim3(static_cast<unsigned>(a.p.blocks), a.p.slices), kFewThreads + 32, smem, s>>>(a);
  if (int e = launched("wgrad_few_kernel")) return e;
  if (a.p.blocks == 1) return 0;
  int sums = a.V * a.C, blocks = static_cast<int>(a.p.blocks), dw_dtype = a.dw_dtype;
  const float* partial = a.partial;
  float scale = a.scale;
  void* dw = a.dw;
  void* args[] = {&partial, &blocks, &sums, &scale, &dw, &dw_dtype};
  return launch_pdl(reinterpret_cast<const void*>(&wgrad_few_join_kernel), dim3((sums + 31) / 32), dim3(1024), 0, s, args, 1,
                    "wgrad_few_join_kernel");
}

template <typename T, typename I, int VEC>
int few_launch_ids(const FewArgs& a, cudaStream_t s) {
  // a predicate and VEC additions per token and row: a kernel for the counts of the networks here, and the most
  if (a.V <= 4) return few_launch_tokens<T, I, VEC, 4>(a, s);
  if (a.V == 5) return few_launch_tokens<T, I, VEC, 5>(a, s);
  return few_launch_tokens<T, I, VEC, kFewTokens>(a, s);
}

template <typename T, int VEC>
int few_launch_vec(const FewArgs& a, cudaStream_t s) {
  return a.id_bytes == 8 ? few_launch_ids<T, int64_t, VEC>(a, s) : few_launch_ids<T, int32_t, VEC>(a, s);
}

template <typename T>
int few_launch(const FewArgs& a, cudaStream_t s) {
  switch (a.p.vec) {
    case 1: return few_launch_vec<T, 1>(a, s);
    case 2: return few_launch_vec<T, 2>(a, s);
    case 4: return few_launch_vec<T, 4>(a, s);
    default:
      if constexpr (sizeof(T) == 2) return few_launch_vec<T, 8>(a, s);
      return fail(BPC_ERR_ARG, "no such vector width");
  }
}

int embed_check(const void* ids, int32_t id_bytes, int64_t n, int32_t V, int32_t C, int64_t stride, int32_t in_dtype,
                int32_t out_dtype) {
  if (n < 0 || n > 0x7fffffffLL || V < 1 || V > 0x7ffffffe || C < 1 || C > (1 << 20))
    return fail(BPC_ERR_ARG, "0 <= n < 2^31 positions, 1 <= V < 2^31 - 1 tokens, 1 <= C <= 2^20 channels");
  if (id_bytes != 4 && id_bytes != 8) return fail(BPC_ERR_ARG, "ids must be int32 or int64 (id_bytes 4 or 8)");
  if (!dtype_size(in_dtype) || !dtype_size(out_dtype)) return fail(BPC_ERR_ARG, "dtype must be f32, bf16 or f16");
  if (stride < C) return fail(BPC_ERR_ARG, "row stride smaller than the channel count");
  if (reinterpret_cast<uintptr_t>(ids) % id_bytes) return fail(BPC_ERR_ARG, "ids are not aligned to their type");
  return 0;
}

}  // namespace

}  // namespace bpc

using namespace bpc;

extern "C" int bpc_embed_lookup(const void* ids, int32_t id_bytes, const void* w, void* y, int64_t n, int32_t V,
                                int32_t C, int64_t w_stride, float scale, int32_t w_dtype, int32_t y_dtype,
                                bpc_stream_t stream) {
  if (int e = embed_check(ids, id_bytes, n, V, C, w_stride, w_dtype, y_dtype)) return e;
  if (n == 0) return 0;
  if (!ids || !w || !y) return fail(BPC_ERR_ARG, "null buffer");
  if (reinterpret_cast<uintptr_t>(w) % dtype_size(w_dtype) || reinterpret_cast<uintptr_t>(y) % dtype_size(y_dtype))
    return fail(BPC_ERR_ARG, "w and y must be aligned to their types");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (id_bytes == 8) return lookup_by_w<int64_t>(ids, w, y, n, V, C, w_stride, scale, w_dtype, y_dtype, s);
  return lookup_by_w<int32_t>(ids, w, y, n, V, C, w_stride, scale, w_dtype, y_dtype, s);
}

extern "C" size_t bpc_embed_wgrad_workspace_size(int64_t n, int32_t V, int32_t C) {
  if (n < 1 || n > 0x7fffffffLL || V < 1 || V > 0x7ffffffe || C < 1 || C > (1 << 20)) return 0;
  return V <= kFewTokens ? few_bytes(n, V, C) : wgrad_plan(n, V, C).bytes;
}

extern "C" int bpc_embed_wgrad(const void* gy, const void* ids, int32_t id_bytes, void* dw, void* workspace,
                               size_t workspace_bytes, int64_t n, int32_t V, int32_t C, int64_t gy_stride, float scale,
                               int32_t gy_dtype, int32_t dw_dtype, bpc_stream_t stream) {
  if (int e = embed_check(ids, id_bytes, n, V, C, gy_stride, gy_dtype, dw_dtype)) return e;
  if (!dw) return fail(BPC_ERR_ARG, "null dw");
  if (reinterpret_cast<uintptr_t>(dw) % dtype_size(dw_dtype)) return fail(BPC_ERR_ARG, "dw must be aligned to its type");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (n == 0) {
    cudaError_t e = cudaMemsetAsync(dw, 0, static_cast<size_t>(V) * C * dtype_size(dw_dtype), s);
    return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string("cudaMemsetAsync: ") + cudaGetErrorString(e));
  }
  if (!gy || !ids || !workspace) return fail(BPC_ERR_ARG, "null buffer");
  if (reinterpret_cast<uintptr_t>(gy) % dtype_size(gy_dtype)) return fail(BPC_ERR_ARG, "gy must be aligned to its type");
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BPC_ERR_ARG, "the workspace must be 16-byte aligned");
  if (workspace_bytes < bpc_embed_wgrad_workspace_size(n, V, C))
    return fail(BPC_ERR_SPACE, "embedding gradient workspace too small");
  if (V <= kFewTokens) {
    FewArgs a;
    a.p = few_plan(gy, dw, n, C, gy_stride, dtype_size(gy_dtype));
    a.gy = gy;
    a.ids = ids;
    a.id_bytes = id_bytes;
    a.n = n;
    a.ldg = gy_stride;
    a.V = V;
    a.C = C;
    a.scale = scale;
    a.dw = dw;
    a.dw_dtype = dw_dtype;
    a.partial = static_cast<float*>(workspace);
    a.status = op_status_ptr();
    if (!a.status) return fail(BPC_ERR_LAUNCH, "cudaGetSymbolAddress(op status) failed");
    if (gy_dtype == BPC_DTYPE_F32) return few_launch<float>(a, s);
    if (gy_dtype == BPC_DTYPE_BF16) return few_launch<__nv_bfloat16>(a, s);
    return few_launch<__half>(a, s);
  }
  const WgradPlan p = wgrad_plan(n, V, C);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int2* const pair[2] = {reinterpret_cast<int2*>(ws + p.pair[0]), reinterpret_cast<int2*>(ws + p.pair[1])};
  int* counts = reinterpret_cast<int*>(ws + p.counts);
  int* totals = reinterpret_cast<int*>(ws + p.totals);
  MergeArgs a;
  const int e =
      id_bytes == 8
          ? sort_ids(static_cast<const int64_t*>(ids), n, V, p, pair, counts, totals, &a.pair, s)
          : sort_ids(static_cast<const int32_t*>(ids), n, V, p, pair, counts, totals, &a.pair, s);
  if (e) return e;
  a.n = n;
  a.items = p.items;
  a.workers = p.workers;
  a.V = V;
  a.C = C;
  a.G = p.G;
  a.ldg = gy_stride;
  a.scale = scale;
  a.dw = dw;
  a.dw_dtype = dw_dtype;
  a.head = reinterpret_cast<float*>(ws + p.head);
  a.tail = reinterpret_cast<float*>(ws + p.tail);
  a.ends = reinterpret_cast<int2*>(ws + p.ends);
  if (gy_dtype == BPC_DTYPE_F32) return merge_launch<float>(gy, a, s);
  if (gy_dtype == BPC_DTYPE_BF16) return merge_launch<__nv_bfloat16>(gy, a, s);
  return merge_launch<__half>(gy, a, s);
}
