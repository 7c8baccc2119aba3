// Linear attention with a decay for each head: a state that forgets at a fixed rate, over whole sequences (forward and
// backward) and one position at a time.
//
//   S_t = a S_(t-1) + k_t v_t^T,   o_t = scale q_t S_t   (a = exp(log_decay_h) per head, S (dk, dv), q, k, v rows)
//
// Forward and every gradient are one scan over rows a_t, b_t, c_t and a state X (da, dc):
//   S = X + in b_t c_t^T;   out_t = out_scale a_t S;   X = a S
//   forward  a, b, c = q, k, v     X = a S_0             out_scale = scale      the last S is the new state
//   dq       a, b, c = go, v, k    X = a S_0^T           out_scale = scale
//   dk       a, b, c = v, go, q    X = gS^T, in = scale  backwards in time      (gS: the gradient of the new state)
//   dv       a, b, c = k, q, go    X = gS, in = scale    backwards in time      a times the last S is dS_0
// A step of the scan takes 32 positions (a chunk) as products of matrices.  With pos the position in the chunk in the
// scan's order, 0 .. r - 1 of r:
//   out_i = out_scale (sum_(pos j <= pos i) in a^(pos i - pos j) (a_i . b_j) c_j + a^(pos i) a_i X)
//   X     = a^r X + sum_j in a^(r - pos j) b_j c_j^T
#include <algorithm>
#include <cmath>
#include <string>

#include "bpc.h"
#include "bpc_common.cuh"
#include "bpc_internal.h"

namespace bpc {

namespace {

constexpr int kThreads = 128;
constexpr int kMaxDim = 128;
constexpr int kChunk = 32;
constexpr int kShort = 16;        // positions that short_kernel takes

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
  float* parts;                 // the segments' states: (B H, segments - 1, da, dc)
  const void* lengths;
  int length_bytes;
  int T, H, da, dc;
  int segments, segment;        // rows per segment, a multiple of kChunk
  uint32_t items;               // B H segments
  float in_scale, out_scale;
  bool first_t, parts_t, vec, out_vec;      // _t: (dc, da)
};

// One scan, or two in one launch (dk and dv): the items of the first, then those of the second
struct Scans {
  Scan s[2];
  uint32_t each, total;
};

__device__ __forceinline__ int length_of(const void* lengths, int bytes, uint32_t b, int T) {
  if (!lengths) return T;
  const int64_t n = bytes == 8 ? static_cast<const int64_t*>(lengths)[b] : static_cast<const int32_t*>(lengths)[b];
  return n < 0 ? 0 : n > T ? T : static_cast<int>(n);
}

// a^n of log2 a, 1 for n = 0 whatever a is (log_decay may be -infinity), 0 for n < 0 (a pair out of order)
__device__ __forceinline__ float log2_decay(const float* log_decay, int h) { return log_decay[h] * 1.4426950408889634f; }
__device__ __forceinline__ float power(float log2_a, int n) {
  float v;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(log2_a * static_cast<float>(n)));
  return n > 0 ? v : n == 0 ? 1.0f : 0.0f;
}

// ---- fragments -------------------------------------------------------------------------------------------------
// mma.sync m16n8k16 (bf16) and m16n8k8 (tf32), fp32 accumulators.  Lane 4 g + t holds of the result rows g, g + 8 and
// columns 2 t, 2 t + 1.  The tf32 products number their k so that lane t's two values are columns 2 t and 2 t + 1 of
// the row-major operand: then an accumulator is an operand of the next product as it stands, and a bf16 operand is one of
// a tf32 product by taking its halves apart.
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ float lds(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float2 lds2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// x = hi + lo in tf32 (11 significant bits), but for 2^-23 of x: hi is x to the nearest, what is left has 12 bits, of which
// a product reads 11.  A NaN may carry over into hi's sign (0x7fffffff makes -0): lo, which is x less that, is NaN then, and so
// it is for infinities and for values from 2^128 (1 - 2^-12) up, which round to infinity.
struct Split {
  uint32_t hi, lo;
  __device__ __forceinline__ explicit Split(float x) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
  }
  Split() = default;
};
// d += a b: three tf32 products leave out the product of the two small parts, 2^-22 of it.  The tensor unit cuts a step's sum off
// where fp32 arithmetic rounds, which adds up along a head: errors of 3.4, 5 to 6, 11 and 20 times 2^-24 of the results' root mean
// square for heads of 16, 32, 64 and 128, where plain fp32 arithmetic makes 1.6 to 3
__device__ __forceinline__ void mma_f32(float (&d)[4], const Split (&a)[4], const Split& b0, const Split& b1) {
  const uint32_t hi[4] = {a[0].hi, a[1].hi, a[2].hi, a[3].hi}, lo[4] = {a[0].lo, a[1].lo, a[2].lo, a[3].lo};
  mma_tf32(d, lo, b0.hi, b1.hi);
  mma_tf32(d, hi, b0.lo, b1.lo);
  mma_tf32(d, hi, b0.hi, b1.hi);
}

// ---- tiles -----------------------------------------------------------------------------------------------------
// 32 rows of DP elements in shared memory.  bf16: 16-byte pieces XORed with the row, so that ldmatrix reads without bank
// conflicts; fp32: rows padded by 16 bytes, so that a lane's reads of four rows and eight columns do.
template <typename T, int DP>
struct Tile {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kCols = DP == 32 ? 32 : 16;                   // of c, per warp: a state of at most 64 values a lane
  static constexpr int kWarps = DP / kCols;                          // of a group, which takes an item
  static constexpr int kThreads = kWarps < 4 ? 128 : 32 * kWarps;
  static constexpr int kGroups = kThreads / 32 / kWarps;
  static constexpr int kMT = kCols / 16;
  static constexpr int kNT = DP / 8;                                 // 8-column pieces of a, b
  static constexpr int kPitch = kF32 ? (DP + 4) * 4 : DP * 2;
  static constexpr int kBytes = kChunk * kPitch;
  static constexpr int kPiece = 16 / sizeof(T);
  static constexpr int kPieces = DP / kPiece;                        // per row
  static constexpr int kStages = kF32 || DP == 32 ? 2 : 3;
  static constexpr int kOutBytes = kF32 ? 0 : 16 * kCols * 2;        // a warp's rows on their way out
  static constexpr int kSmem = kGroups * kStages * 3 * kBytes + kGroups * kWarps * kOutBytes;
  static constexpr int kBlocks = kWarps == 8 ? 1 : kSmem > 74 * 1024 || DP == 32 ? 2 : 3;      // per SM: registers and shared memory
  __device__ static __forceinline__ uint32_t at(int row, int piece) {
    if constexpr (kF32) return row * kPitch + piece * 16;
    else return row * kPitch + ((piece ^ (DP == 16 ? row >> 2 & 1 : DP == 32 ? row >> 1 & 3 : row & 7)) << 4);
  }
};

__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows [0, rows) of `src` (row stride in elements) into a tile, zeros behind them and behind dim; by one group of warps
template <typename T, int DP>
__device__ __forceinline__ void load_tile(uint32_t tile, const T* src, int64_t stride, int rows, int dim, bool vec, int lane) {
  using L = Tile<T, DP>;
  constexpr int kLanes = 32 * L::kWarps, kPasses = kChunk * L::kPieces / kLanes, kStep = kLanes / L::kPieces;      // rows per pass
  if (vec) {
    static_assert(kLanes % L::kPieces == 0, "a lane keeps its piece of a row");
    const int row = lane / L::kPieces, piece = lane % L::kPieces;
    const T* at = src + row * stride + piece * L::kPiece;
    const bool inside = piece * L::kPiece < dim;
#pragma unroll
    for (int k = 0; k < kPasses; ++k) {
      const bool there = inside && row + k * kStep < rows;
      cp_async(tile + L::at(row + k * kStep, piece), there ? at : src, there ? 16 : 0);
      at += kStep * stride;
    }
  } else {
    for (int e = lane; e < kChunk * DP; e += kLanes) {
      const int row = e / DP, col = e % DP;
      const T v = row < rows && col < dim ? src[row * stride + col] : T(0.0f);
      const uint32_t dst = tile + L::at(row, col / L::kPiece) + col % L::kPiece * sizeof(T);
      if constexpr (L::kF32) asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst), "f"(v) : "memory");
      else asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst), "h"(__bfloat16_as_ushort(v)) : "memory");
    }
  }
}

// ---- a chunk ---------------------------------------------------------------------------------------------------
// A chunk is worked on in halves of 16 rows, in the scan's order: half 0 is the rows 0 - 15 forwards, 16 - 31 backwards (where
// the chunk has more than 16 rows).  A lane's weights: of pairs of positions whose 8-row pieces are D = 0 .. 3 apart in
// the scan's order (columns 2 t, 2 t + 1 of them); of the state for rows g, g + 8 of a half; of c's rows 2 t, 2 t + 1, 2 t + 8,
// 2 t + 9 of a half in the state's update; of the state there.
template <bool REV>
struct Weights {
  float pair[4][2], row[2][2], update[2][4], keep;
  bool in_order[2];             // D = 0: the columns 2 t, 2 t + 1 that do not come after the row
  int halves, flip;             // flip: half 0 is rows 16 - 31

  // r: the chunk's rows; until: the position as of which the state is wanted, r or (as of the last one) r - 1
  __device__ __forceinline__ void of_pairs(float log2_a, float in) {
    const int lane = threadIdx.x & 31, e0 = (lane >> 2) - 2 * (lane & 3);
#pragma unroll
    for (int D = 0; D < 4; ++D)
#pragma unroll
      for (int z = 0; z < 2; ++z) pair[D][z] = in * power(log2_a, 8 * D + (REV ? z - e0 : e0 - z));
#pragma unroll
    for (int z = 0; z < 2; ++z) in_order[z] = (REV ? z - e0 : e0 - z) >= 0;
  }
  __device__ __forceinline__ void of_rows(float log2_a, float in, int r, int until) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    halves = r > 16 ? 2 : 1;
    flip = REV && halves == 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row0 = (flip ? 1 - h : h) * 16;
#pragma unroll
      for (int k = 0; k < 2; ++k) row[h][k] = power(log2_a, REV ? r - 1 - (row0 + g + 8 * k) : row0 + g + 8 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = row0 + 2 * t + (k & 1) + (k >> 1) * 8;
        update[h][k] = in * power(log2_a, until - (REV ? r - 1 - j : j));
      }
    }
    keep = power(log2_a, until);
  }
  // the product of a pair in 8-row pieces i and j of their halves, column z: weighed, and dropped (not multiplied by zero)
  // where j comes after i
  __device__ __forceinline__ float weigh(float p, int i_half, int j_half, int i, int j, int z) const {
    const int D = 2 * (i_half - j_half) + (REV ? j - i : i - j);
    return D < 0 || (D == 0 && !in_order[z]) ? 0.0f : p * pair[D < 0 ? 0 : D][z];
  }
};

template <typename T, int DP, bool REV>
struct Warp {
  using L = Tile<T, DP>;
  static constexpr int kMT = L::kMT, kNT = L::kNT;
  float X[kMT][kNT][4];         // X^T: rows = this warp's columns of c, columns = those of a, b

  // O (16 positions x this warp's columns of c, for each half), and X after the chunk.  SPLIT: bf16 parts of the weighted c.
  // FULL: more than 16 rows, a state and an update, as nearly all chunks of long sequences; their many branches cost as much
  // again as the products.
  template <bool OUT, int SPLIT>
  __device__ __forceinline__ void chunk(uint32_t sa, uint32_t sb, uint32_t sc, int slice, const Weights<REV>& w, bool use_x,
                                        bool update, float (&O)[2][2 * kMT][4]) {
    if (w.halves == 2 && use_x && update) chunk_of<true, OUT, SPLIT>(sa, sb, sc, slice, w, true, true, O);
    else chunk_of<false, OUT, SPLIT>(sa, sb, sc, slice, w, use_x, update, O);
  }
  template <bool FULL, bool OUT, int SPLIT>
  __device__ __forceinline__ void chunk_of(uint32_t sa, uint32_t sb, uint32_t sc, int slice, const Weights<REV>& w, bool use_x,
                                           bool update, float (&O)[2][2 * kMT][4]) {
    if constexpr (L::kF32) chunk_f32<FULL, OUT>(sa, sb, sc, slice, w, use_x, update, O);
    else chunk_bf16<FULL, OUT, SPLIT>(sa, sb, sc, slice, w, use_x, update, O);
  }

  // What is fp32 and an operand of a bf16 product (the weighted a b^T, X, the weighted c) goes in as two bf16 parts, off by
  // at most 2^-18 of itself; one part would round as coarsely as the result.  Where a state is handed out, c as three.  A value
  // that is not finite, or rounds to infinity in its first part (2^128 (1 - 2^-9) and more), has a second part of NaN.
  template <bool FULL, bool OUT, int SPLIT>
  __device__ __forceinline__ void chunk_bf16(uint32_t sa, uint32_t sb, uint32_t sc, int slice, const Weights<REV>& w, bool use_x,
                                             bool update, float (&O)[2][2 * kMT][4]) {
    constexpr int kKS = DP / 16;
    const int lane = threadIdx.x & 31;
    // addresses of a lane's row in four 8 x 8 pieces: row lane % 16 and column piece lane / 16, or (b as the second
    // operand of a b^T) row lane % 8 + 8 (lane / 16) and column piece lane / 8 % 2; the next 16 columns are an XOR by 32
    const uint32_t by_row = L::at(lane & 15, lane >> 4), by_piece = L::at((lane & 7) + (lane >> 4) * 8, lane >> 3 & 1);
    const uint32_t half[2] = {w.flip ? 16u * L::kPitch : 0u, w.flip ? 0u : 16u * L::kPitch};
    const bool two = FULL || w.halves == 2;
    uint32_t c[2][kMT][4];
    {
      const uint32_t c0 = L::at(lane & 15, slice * (L::kCols / 8) + (lane >> 4));
#pragma unroll
      for (int m = 0; m < kMT; ++m) ldmatrix_trans(c[0][m], sc + half[0] + (c0 ^ (m << 5)));
      if (two) {
#pragma unroll
        for (int m = 0; m < kMT; ++m) ldmatrix_trans(c[1][m], sc + half[1] + (c0 ^ (m << 5)));
      }
    }
    if constexpr (OUT) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 2 * kMT; ++n) O[h][n][0] = O[h][n][1] = O[h][n][2] = O[h][n][3] = 0.0f;
      float P[3][2][4] = {};                       // halves (0, 0), (1, 0), (1, 1)
#pragma unroll
      for (int k = 0; k < kKS; ++k) {
        uint32_t a[2][4], b[4];
        ldmatrix(a[0], sa + half[0] + (by_row ^ (k << 5)));
        ldmatrix(b, sb + half[0] + (by_piece ^ (k << 5)));
        mma_bf16(P[0][0], a[0], b[0], b[1]);
        mma_bf16(P[0][1], a[0], b[2], b[3]);
        if (two) {
          ldmatrix(a[1], sa + half[1] + (by_row ^ (k << 5)));
          mma_bf16(P[1][0], a[1], b[0], b[1]);
          mma_bf16(P[1][1], a[1], b[2], b[3]);
          ldmatrix(b, sb + half[1] + (by_piece ^ (k << 5)));
          mma_bf16(P[2][0], a[1], b[0], b[1]);
          mma_bf16(P[2][1], a[1], b[2], b[3]);
        }
        if (FULL || use_x) {
#pragma unroll
          for (int n = 0; n < 2 * kMT; ++n) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const float x0 = X[n / 2][2 * k + z][2 * (n % 2)], x1 = X[n / 2][2 * k + z][2 * (n % 2) + 1];
              hi[z] = pack(x0, x1);
              lo[z] = pack(x0 - low(hi[z]), x1 - high(hi[z]));
            }
            mma_bf16(O[0][n], a[0], lo[0], lo[1]);
            mma_bf16(O[0][n], a[0], hi[0], hi[1]);
            if (two) {
              mma_bf16(O[1][n], a[1], lo[0], lo[1]);
              mma_bf16(O[1][n], a[1], hi[0], hi[1]);
            }
          }
        }
      }
      if (FULL || use_x) weigh_rows(w, O);
#pragma unroll
      for (int block = 0; block < 3; ++block) {
        const int i_half = block > 0, j_half = block > 1;
        if (block == 0 || two) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {            // (rows g, columns of piece 0), (g + 8, 0), (g, 1), (g + 8, 1)
            const int r = e & 1, n = e >> 1;
            const float p0 = w.weigh(P[block][n][2 * r], i_half, j_half, r, n, 0);
            const float p1 = w.weigh(P[block][n][2 * r + 1], i_half, j_half, r, n, 1);
            hi[e] = pack(p0, p1);
            lo[e] = pack(p0 - low(hi[e]), p1 - high(hi[e]));
          }
#pragma unroll
          for (int n = 0; n < 2 * kMT; ++n) {
            const uint32_t b0 = c[j_half][n / 2][2 * (n % 2)], b1 = c[j_half][n / 2][2 * (n % 2) + 1];
            mma_bf16(O[i_half][n], lo, b0, b1);
            mma_bf16(O[i_half][n], hi, b0, b1);
          }
        }
      }
    }
    if (FULL || update) {
      uint32_t wc[2][SPLIT][kMT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (h == 0 || two) {
#pragma unroll
          for (int m = 0; m < kMT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {          // c's pieces: (positions 0-7, columns 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
              const int to = (e & 1) * 2 + (e >> 1);         // their places in the transposed first operand
              float x0 = low(c[h][m][e]) * w.update[h][2 * (e & 1)], x1 = high(c[h][m][e]) * w.update[h][2 * (e & 1) + 1];
#pragma unroll
              for (int s = 0; s < SPLIT; ++s) {
                wc[h][s][m][to] = pack(x0, x1);
                x0 -= low(wc[h][s][m][to]), x1 -= high(wc[h][s][m][to]);
              }
            }
        }
#pragma unroll
      for (int k = 0; k < kKS; ++k) {
        uint32_t b[2][4];
        ldmatrix_trans(b[0], sb + half[0] + (by_row ^ (k << 5)));
        if (two) ldmatrix_trans(b[1], sb + half[1] + (by_row ^ (k << 5)));
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            float u[4] = {};
#pragma unroll
            for (int s = SPLIT - 1; s >= 0; --s) mma_bf16(u, wc[0][s][m], b[0][2 * z], b[0][2 * z + 1]);
            if (two) {
#pragma unroll
              for (int s = SPLIT - 1; s >= 0; --s) mma_bf16(u, wc[1][s][m], b[1][2 * z], b[1][2 * z + 1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) X[m][2 * k + z][e] = fmaf(w.keep, X[m][2 * k + z][e], u[e]);
          }
      }
    }
  }

  __device__ static __forceinline__ void weigh_rows(const Weights<REV>& w, float (&O)[2][2 * kMT][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < 2 * kMT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[h][n][e] *= w.row[h][e >> 1];
  }

  template <bool FULL, bool OUT>
  __device__ __forceinline__ void chunk_f32(uint32_t sa, uint32_t sb, uint32_t sc, int slice, const Weights<REV>& w, bool use_x,
                                            bool update, float (&O)[2][2 * kMT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t half[2] = {w.flip ? 16u * L::kPitch : 0u, w.flip ? 0u : 16u * L::kPitch};
    const bool two = FULL || w.halves == 2;
    const uint32_t pair_at = g * L::kPitch + t * 8;              // (row g, columns 2 t, 2 t + 1)
    const uint32_t cross_at = 2 * t * L::kPitch + g * 4;         // (rows 2 t and the next, column g)
    const uint32_t c0 = sc + cross_at + slice * (L::kCols * 4);
    if constexpr (OUT) {
      float P[3][2][4] = {};                       // halves (0, 0), (1, 0), (1, 1)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 2 * kMT; ++n) O[h][n][0] = O[h][n][1] = O[h][n][2] = O[h][n][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < kNT; ++k) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (h == 0 || two) {
            const float2 a0 = lds2(sa + half[h] + pair_at + k * 32), a1 = lds2(sa + half[h] + pair_at + 8 * L::kPitch + k * 32);
            const Split a[4] = {Split(a0.x), Split(a1.x), Split(a0.y), Split(a1.y)};
#pragma unroll
            for (int j = 0; j <= h; ++j)
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float2 b = lds2(sb + half[j] + pair_at + n * 8 * L::kPitch + k * 32);
                mma_f32(P[h + j][n], a, Split(b.x), Split(b.y));
              }
            if (FULL || use_x) {
#pragma unroll
              for (int n = 0; n < 2 * kMT; ++n)
                mma_f32(O[h][n], a, Split(X[n / 2][k][2 * (n % 2)]), Split(X[n / 2][k][2 * (n % 2) + 1]));
            }
          }
      }
      if (FULL || use_x) weigh_rows(w, O);
#pragma unroll
      for (int block = 0; block < 3; ++block) {
        const int i_half = block > 0, j_half = block > 1;
        if (block == 0 || two) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {            // 8 positions j at a time
            Split p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)            // (g, 2 t), (g + 8, 2 t), (g, 2 t + 1), (g + 8, 2 t + 1)
              p[e] = Split(w.weigh(P[block][k][2 * (e & 1) + (e >> 1)], i_half, j_half, e & 1, k, e >> 1));
            const uint32_t at = c0 + half[j_half] + k * 8 * L::kPitch;
#pragma unroll
            for (int n = 0; n < 2 * kMT; ++n)
              mma_f32(O[i_half][n], p, Split(lds(at + n * 32)), Split(lds(at + L::kPitch + n * 32)));
          }
        }
      }
    }
    if (FULL || update) {
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        float u[kNT][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (h == 0 || two) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t rows = half[h] + k * 8 * L::kPitch;
              Split wc[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)          // (column g, 2 t), (g + 8, 2 t), (g, 2 t + 1), (g + 8, 2 t + 1)
                wc[e] = Split(w.update[h][2 * k + (e >> 1)] * lds(c0 + rows + (e >> 1) * L::kPitch + (2 * m + (e & 1)) * 32));
#pragma unroll
              for (int n = 0; n < kNT; ++n)
                mma_f32(u[n], wc, Split(lds(sb + rows + cross_at + n * 32)), Split(lds(sb + rows + cross_at + L::kPitch + n * 32)));
            }
          }
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) X[m][n][e] = fmaf(w.keep, X[m][n][e], u[n][e]);
      }
    }
  }

  // f(value of X, column of a, column of c) over a lane's values
  template <typename F>
  __device__ __forceinline__ void each(int slice, F f) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f(X[m][n][e], n * 8 + 2 * (lane & 3) + (e & 1), slice * L::kCols + m * 16 + (lane >> 2) + (e >> 1) * 8);
  }
};

// ---- an item: a sequence's head, or one segment of it ------------------------------------------------------------
struct Item {
  uint32_t b;
  int h, segment, n;            // n: the sequence's length
  int row0, rows;               // its first row, its valid rows
  int steps;                    // chunks with valid rows, one at least
  __device__ __forceinline__ Item(const Scan& p, uint32_t at) {
    const uint32_t rest = at / p.H;
    h = static_cast<int>(at - rest * p.H);
    b = p.segments > 1 ? rest / p.segments : rest;
    segment = p.segments > 1 ? static_cast<int>(rest - b * p.segments) : 0;
    n = length_of(p.lengths, p.length_bytes, b, p.T);
    row0 = segment * p.segment;
    const int left = n - row0;
    rows = left < 0 ? 0 : left > p.segment ? p.segment : left;
    steps = rows ? (rows + kChunk - 1) / kChunk : 1;
  }
  __device__ __forceinline__ int valid(int c) const { return rows - c * kChunk < kChunk ? rows - c * kChunk : kChunk; }
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& r, const Item& it, int row) {
  return static_cast<const T*>(r.at) + it.b * r.b + row * r.t + it.h * r.h;
}

// 16 rows of a warp's output columns, zeros from row `rows` on; rows behind `until` stay
template <typename T, int DP>
__device__ __forceinline__ void store_rows(T* out, int64_t stride, const float (&O)[2 * Tile<T, DP>::kMT][4], int slice, int rows,
                                           int until, int dc, float scale, bool vec, uint32_t stage) {
  using L = Tile<T, DP>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int kCols = L::kCols;
  out += slice * kCols;
  dc -= slice * kCols;
  if (!vec) {
#pragma unroll
    for (int n = 0; n < 2 * L::kMT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = g + (e >> 1) * 8, col = n * 8 + 2 * t + (e & 1);
        if (row < until && col < dc) store_f32(out + row * stride + col, row < rows ? scale * O[n][e] : 0.0f);
      }
  } else if constexpr (L::kF32) {
#pragma unroll
    for (int n = 0; n < 2 * L::kMT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = g + e * 8, col = n * 8 + 2 * t;
        if (row < until && col < dc)
          *reinterpret_cast<float2*>(out + row * stride + col) =
              row < rows ? make_float2(scale * O[n][2 * e], scale * O[n][2 * e + 1]) : make_float2(0.0f, 0.0f);
      }
  } else {
    // through shared memory: whole rows of 64 (32) bytes, of which a quad alone has 16
    __syncwarp();
#pragma unroll
    for (int n = 0; n < 2 * L::kMT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = g + e * 8;
        const uint32_t v = row < rows ? pack(scale * O[n][2 * e], scale * O[n][2 * e + 1]) : 0u;
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + row * kCols * 2 + ((n ^ (row >> 1 & (2 * L::kMT - 1))) << 4) + t * 4), "r"(v)
                     : "memory");
      }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < L::kMT; ++k) {
      const int e = k * 32 + lane, row = e / (2 * L::kMT), n = e % (2 * L::kMT);
      uint4 v;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "r"(stage + row * kCols * 2 + ((n ^ (row >> 1 & (2 * L::kMT - 1))) << 4))
                   : "memory");
      if (row < until && n * 8 < dc) *reinterpret_cast<uint4*>(out + row * stride + n * 8) = v;
    }
  }
}

// Rows [from, to) of a warp's output columns become zero
template <typename T, int DP>
__device__ __forceinline__ void zero_rows(T* out, int64_t stride, int slice, int from, int to, int dc) {
  const int lane = threadIdx.x & 31, first = slice * Tile<T, DP>::kCols;
  if (lane >= min(dc - first, Tile<T, DP>::kCols)) return;
  for (int row = from; row < to; ++row) store_f32(out + row * stride + first + lane, 0.0f);
}

// A group of warps takes an item at a time, chunk by chunk, each warp some columns of c; the state stays in the warps'
// registers.  Twelve warps an SM, whose dependent products and conversions bound it: 30,011 positions x 12 bf16 heads of 64
// take 85 us (184 MB: 28 at the copy's rate), the tensor unit 40 % busy, 0.48 instructions a cycle and scheduler.  16
// columns a warp and three blocks an SM against 32 and two: 115 us.  Chunks of 16 positions read and cut the state twice as
// often; the state read as tf32 (11 bits) would save the cutting, and show in the result.  The tiles of the next chunks, of
// the next items too, are on their way meanwhile.  REV: backwards in time.
// OUT false: the states that the segments leave behind alone.
template <typename T, int DP, bool REV, bool OUT, int SPLIT>
__global__ void __launch_bounds__(Tile<T, DP>::kThreads, Tile<T, DP>::kBlocks) scan_kernel(const __grid_constant__ Scans all) {
  using L = Tile<T, DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kS = L::kStages;
  const int warp = threadIdx.x >> 5, group = warp / L::kWarps, slice = warp % L::kWarps;
  const int lane_in_group = threadIdx.x - group * (32 * L::kWarps);
  const uint32_t base = smem_u32(smem) + group * (kS * 3 * L::kBytes);
  const uint32_t stage_out = smem_u32(smem) + L::kGroups * (kS * 3 * L::kBytes) + warp * L::kOutBytes;
  const uint32_t first_item = blockIdx.x * L::kGroups + group, stride = gridDim.x * L::kGroups;
  auto sync = [&] {
    if constexpr (L::kWarps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * L::kWarps) : "memory");
  };

  // the loads' item, its chunk's rows and its steps left
  uint32_t ahead_at = first_item, ahead_tile = base;
  const T *ahead_a = nullptr, *ahead_b = nullptr, *ahead_c = nullptr;
  int ahead_left = 0, ahead_r = 0;
  const int64_t by = REV ? -kChunk : kChunk;
  // two scans backwards only, as dk and dv: to ask which one it is costs the others a quarter (16,384 rounds 63 -> 80 us)
  auto scan_of = [&](uint32_t at) { return &all.s[REV && OUT && at >= all.each ? 1 : 0]; };
  const Scan* ahead_p = all.s;
  auto start = [&] {
    ahead_p = scan_of(ahead_at);
    const Scan& p = *ahead_p;
    const Item it(p, ahead_at - (ahead_p == all.s ? 0 : all.each));
    ahead_left = it.steps;
    const int c = REV ? it.steps - 1 : 0, row = it.row0 + c * kChunk;
    ahead_r = it.rows - (REV ? c * kChunk : 0);      // backwards the first chunk may be short, forwards the last
    ahead_a = row_of<T>(p.a, it, row), ahead_b = row_of<T>(p.b, it, row), ahead_c = row_of<T>(p.c, it, row);
  };
  if (ahead_at < all.total) start();
  auto load = [&] {
    if (ahead_at < all.total) {
      const Scan& p = *ahead_p;
      const int r = min(ahead_r, kChunk);
      if constexpr (OUT) load_tile<T, DP>(ahead_tile, ahead_a, p.a.t, r, p.da, p.vec, lane_in_group);
      load_tile<T, DP>(ahead_tile + L::kBytes, ahead_b, p.b.t, r, p.da, p.vec, lane_in_group);
      load_tile<T, DP>(ahead_tile + 2 * L::kBytes, ahead_c, p.c.t, r, p.dc, p.vec, lane_in_group);
      ahead_a += by * p.a.t, ahead_b += by * p.b.t, ahead_c += by * p.c.t;
      ahead_r = REV ? kChunk : ahead_r - kChunk;
      if (--ahead_left == 0) {
        ahead_at += stride;
        if (ahead_at < all.total) start();
      }
    }
    ahead_tile = ahead_tile == base + (kS - 1) * (3 * L::kBytes) ? base : ahead_tile + 3 * L::kBytes;
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < kS - 1; ++s) load();
  // the kernels of one call follow one another programmatically: the inputs were there before the first, the states are when
  // the one before is done
  if constexpr (!OUT) pdl_launch_dependents();
  else pdl_wait();

  Warp<T, DP, REV> state;
  uint32_t tile = base;
  for (uint32_t at = first_item; at < all.total; at += stride) {
    const Scan& p = *scan_of(at);
    const Item it(p, at - (&p == all.s ? 0 : all.each));
    const int64_t bh = static_cast<int64_t>(it.b) * p.H + it.h;
    const float log2_a = log2_decay(p.log_decay, it.h);
    // where the scan enters and leaves the sequence
    const int end_segment = (it.n ? it.n - 1 : 0) / p.segment;
    const bool enters = it.segment == (REV ? end_segment : 0), leaves = it.segment == (REV ? 0 : end_segment);
    const bool beyond = it.segment > end_segment;
    const float* f = nullptr;                      // what X starts from
    float lead = 1.0f;
    bool turned = p.first_t;
    if (enters) {
      if (p.first) f = p.first + bh * p.da * p.dc;
      if (!REV && it.n) lead = power(log2_a, 1);
    } else if (OUT && !beyond) {
      f = p.parts + (bh * (p.segments - 1) + (REV ? it.segment : it.segment - 1)) * (p.da * p.dc);
      turned = p.parts_t;
    }
    state.each(slice, [&](float& x, int i, int j) {
      x = f && i < p.da && j < p.dc ? lead * f[turned ? j * p.da + i : i * p.dc + j] : 0.0f;
    });
    bool use_x = f != nullptr;
    const bool keeps = OUT ? leaves && p.last : true;
    Weights<REV> w;
    if constexpr (OUT) w.of_pairs(log2_a, p.in_scale);
    int weights_r = -1, weights_until = -1;
    const int64_t out_stride = static_cast<int64_t>(p.H) * p.dc;
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(it.b) * p.T * p.H + it.h) * p.dc;
    for (int step = 0; step < it.steps; ++step) {
      const int c = REV ? it.steps - 1 - step : step, row = it.row0 + c * kChunk, r = it.valid(c);
      const bool final = step + 1 == it.steps;
      // forwards the state that is handed out is as of the last position, without the decay into the next
      const int until = OUT && !REV && final && keeps ? (r ? r - 1 : 0) : r;
      if (r != weights_r || until != weights_until) {
        w.of_rows(log2_a, p.in_scale, r, until);
        weights_r = r, weights_until = until;
      }
      cp_wait<kS - 2>();
      sync();
      load();
      float O[2][2 * L::kMT][4];
      state.template chunk<OUT, SPLIT>(tile, tile + L::kBytes, tile + 2 * L::kBytes, slice, w, use_x, !final || keeps, O);
      tile = tile == base + (kS - 1) * (3 * L::kBytes) ? base : tile + 3 * L::kBytes;
      if constexpr (OUT) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int from = (w.flip ? 1 - h : h) * 16;
          if (h < w.halves)
            store_rows<T, DP>(out + (row + from) * out_stride, out_stride, O[h], slice, r - from, p.T - row - from, p.dc,
                              p.out_scale, p.out_vec, stage_out);
        }
        if (w.halves == 1) zero_rows<T, DP>(out, out_stride, slice, row + 16, min(p.T, row + kChunk), p.dc);
      }
      use_x = true;
    }
    if constexpr (OUT) {
      zero_rows<T, DP>(out, out_stride, slice, it.row0 + it.steps * kChunk, min(p.T, it.row0 + p.segment), p.dc);
      if (keeps) {
        float* to = p.last + bh * p.da * p.dc;
        state.each(slice, [&](float& x, int i, int j) {
          if (i < p.da && j < p.dc) to[i * p.dc + j] = x;
        });
      }
    } else if (it.segment != (REV ? 0 : p.segments - 1)) {
      float* to = p.parts + (bh * (p.segments - 1) + (REV ? it.segment - 1 : it.segment)) * (p.da * p.dc);
      state.each(slice, [&](float& x, int i, int j) {
        if (i < p.da && j < p.dc) to[i * p.dc + j] = x;
      });
    }
  }
}

// The states that the segments leave behind, alone, become those that their next ones start from: a thread per value of
// a state, along the segments.
template <bool REV>
__global__ void __launch_bounds__(256) join_kernel(const Scan p, int per) {      // blocks per state
  const uint32_t bh = blockIdx.x / per;
  const int b = bh / p.H, n = length_of(p.lengths, p.length_bytes, b, p.T), D = p.da * p.dc;
  const int e = blockIdx.x % per * 256 + threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if (e >= D) return;
  const float log2_a = log2_decay(p.log_decay, bh - b * p.H);
  float* f = p.parts + static_cast<int64_t>(bh) * (p.segments - 1) * D + e;
  float x = 0.0f;
  constexpr int kAhead = 32;
  for (int s0 = 0; s0 < p.segments - 1; s0 += kAhead) {
    float v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int s = REV ? p.segments - 2 - s0 - u : s0 + u;
      v[u] = s0 + u < p.segments - 1 ? f[static_cast<int64_t>(s) * D] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s0 + u < p.segments - 1) {
        const int s = REV ? p.segments - 2 - s0 - u : s0 + u;
        const int left = n - (REV ? s + 1 : s) * p.segment;
        x = fmaf(power(log2_a, left < 0 ? 0 : left > p.segment ? p.segment : left), x, v[u]);
        f[static_cast<int64_t>(s) * D] = x;
      }
    }
  }
}

// ---- short sequences ---------------------------------------------------------------------------------------------
// Up to 16 positions and no state: out_i = scale sum_(j <= i) a^(i - j) (a_i . b_j) c_j (j >= i for dk and dv), one warp
// per sequence and head, in registers.  A lane loads 16-byte pieces of rows g and g + 8.  The sum over a's columns may
// number them as it likes, so a piece's words are operands as they lie; c's 8 x 8 pieces are transposed by the tensor
// unit's move; and a result's columns come out where c's pieces had them, so that a lane stores the pieces it would load.
// The forward pass reads three and writes one tensor, the backward pass reads four and writes three: no state, and nothing
// twice.  Up to 8 positions (HALVES 1) take half of the work: 25,600 heads of 5 fp32 positions 31 -> 20 us, 18 with splits of one addition less.
//   bf16 heads of 32 are bound by memory: 371,712 of 11 positions 182 us forwards (5.8 TB/s of 1.05 GB), 343 backwards (5.3 of
// 1.84).  Through shared memory and the long sequences' kernel, at 833 instructions a head against 240, they took 500 us a scan;
// a state's worth of registers cost the occupancy that hides the loads.
struct Short {
  Rows q, k, v, go;
  void *o, *dq, *dk, *dv;       // o, or the gradients
  const float* log_decay;
  const void* lengths;
  int length_bytes, T, H, dim_k, dim_v;
  float scale;
  uint32_t items, step_b, step_h;     // B H; a grid's warps as sequences and heads
};

template <typename T, int DP, int HALVES>
struct Piece {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kWords = DP * static_cast<int>(sizeof(T)) / 16;      // of a lane, per row
  static constexpr int kWide = kWords < 4 ? kWords : 4;                    // of a load
  static constexpr int kElements = kWide * 4 / static_cast<int>(sizeof(T));
  uint32_t r[HALVES][kWords];
  // column of a lane's first element of load k
  __device__ static __forceinline__ int column(int k) { return k * 4 * kElements + (threadIdx.x & 3) * kElements; }

  __device__ __forceinline__ void load(const T* row, int64_t stride, int rows, int dim) {
    const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int k = 0; k < kWords / kWide; ++k) {
        const bool there = g + 8 * h < rows && column(k) < dim;
        const T* at = row + (g + 8 * h) * stride + column(k);
        if constexpr (kWide == 4) {
          const uint4 v = there ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
          r[h][4 * k] = v.x, r[h][4 * k + 1] = v.y, r[h][4 * k + 2] = v.z, r[h][4 * k + 3] = v.w;
        } else {
          const uint2 v = there ? __ldg(reinterpret_cast<const uint2*>(at)) : make_uint2(0, 0);
          r[h][2 * k] = v.x, r[h][2 * k + 1] = v.y;
        }
      }
  }
  __device__ __forceinline__ void store(T* row, int64_t stride, int until, int dim) const {
    const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int k = 0; k < kWords / kWide; ++k) {
        T* at = row + (g + 8 * h) * stride + column(k);
        if (g + 8 * h < until && column(k) < dim) {
          if constexpr (kWide == 4)
            *reinterpret_cast<uint4*>(at) = make_uint4(r[h][4 * k], r[h][4 * k + 1], r[h][4 * k + 2], r[h][4 * k + 3]);
          else *reinterpret_cast<uint2*>(at) = make_uint2(r[h][2 * k], r[h][2 * k + 1]);
        }
      }
  }
};

__device__ __forceinline__ uint32_t transpose(uint32_t piece) {      // an 8 x 8 piece of 16-bit elements
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(piece));
  return r;
}

// weights of (i, j): w[0], w[1] for i and j in the same half of the positions, w[2], w[3] for the later half's with the
// earlier one's
struct PairWeights {
  float w[4];
  bool in_order[2];             // of the same half: the columns that do not come after the row
  __device__ __forceinline__ PairWeights(float log2_a, bool reverse, float scale) {
    const int lane = threadIdx.x & 31, e0 = (lane >> 2) - 2 * (lane & 3);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = scale * power(log2_a, (reverse ? (k & 1) - e0 : e0 - (k & 1)) + (k >> 1) * 8);
#pragma unroll
    for (int k = 0; k < 2; ++k) in_order[k] = (reverse ? k - e0 : e0 - k) >= 0;
  }
};

template <typename T, int DP, int HALVES>
__device__ __forceinline__ Piece<T, DP, HALVES> attend(const Piece<T, DP, HALVES>& a, const Piece<T, DP, HALVES>& b,
                                                       const Piece<T, DP, HALVES>& c, const PairWeights& w, bool reverse, int rows) {
  using P_ = Piece<T, DP, HALVES>;
  constexpr int kLast = HALVES - 1;
  auto second = [](uint32_t x) { return HALVES == 2 ? x : 0u; };      // of rows g + 8
  const int g = (threadIdx.x & 31) >> 2;
  float P[HALVES][4] = {};
  P_ out;
  if constexpr (P_::kF32) {
#pragma unroll
    for (int k = 0; k < P_::kWords / 2; ++k) {
      const Split x[4] = {Split(__uint_as_float(a.r[0][2 * k])), Split(__uint_as_float(second(a.r[kLast][2 * k]))),
                          Split(__uint_as_float(a.r[0][2 * k + 1])), Split(__uint_as_float(second(a.r[kLast][2 * k + 1])))};
#pragma unroll
      for (int n = 0; n < HALVES; ++n)
        mma_f32(P[n], x, Split(__uint_as_float(b.r[n][2 * k])), Split(__uint_as_float(b.r[n][2 * k + 1])));
    }
  } else {
#pragma unroll
    for (int k = 0; k < P_::kWords / 2; ++k) {
      const uint32_t x[4] = {a.r[0][2 * k], second(a.r[kLast][2 * k]), a.r[0][2 * k + 1], second(a.r[kLast][2 * k + 1])};
#pragma unroll
      for (int n = 0; n < HALVES; ++n) mma_bf16(P[n], x, b.r[n][2 * k], b.r[n][2 * k + 1]);
    }
  }
  // [n][row half][column]: products out of order are dropped, not multiplied by zero; others are multiplied whatever their
  // weight is, for a NaN shows through a weight of zero too
#pragma unroll
  for (int n = 0; n < HALVES; ++n)
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const bool ordered = h == n ? w.in_order[z] : reverse ? h < n : n < h;
        float& x = P[n][2 * h + z];
        x = ordered ? x * w.w[h == n ? z : 2 + z] : 0.0f;
      }
  const bool keep0 = g < rows, keep1 = g + 8 < rows;
  if constexpr (P_::kF32) {
    Split p[HALVES][4];
#pragma unroll
    for (int n = 0; n < HALVES; ++n) {
      p[n][0] = Split(P[n][0]), p[n][1] = Split(HALVES == 2 ? P[n][2] : 0.0f);
      p[n][2] = Split(P[n][1]), p[n][3] = Split(HALVES == 2 ? P[n][3] : 0.0f);
    }
#pragma unroll
    for (int q = 0; q < P_::kWords / 2; ++q) {
      float O[4] = {};
#pragma unroll
      for (int n = 0; n < HALVES; ++n) {
        // 32-bit elements as two pieces of 16-bit ones
        const uint32_t x0 = c.r[n][2 * q], x1 = c.r[n][2 * q + 1];
        const uint32_t lo = transpose(__byte_perm(x0, x1, 0x5410)), hi = transpose(__byte_perm(x0, x1, 0x7632));
        mma_f32(O, p[n], Split(__uint_as_float(__byte_perm(lo, hi, 0x5410))), Split(__uint_as_float(__byte_perm(lo, hi, 0x7632))));
      }
      out.r[0][2 * q] = keep0 ? __float_as_uint(O[0]) : 0u, out.r[0][2 * q + 1] = keep0 ? __float_as_uint(O[1]) : 0u;
      if (HALVES == 2)
        out.r[kLast][2 * q] = keep1 ? __float_as_uint(O[2]) : 0u, out.r[kLast][2 * q + 1] = keep1 ? __float_as_uint(O[3]) : 0u;
    }
  } else {
    // the weighted products as two bf16 parts, off by 2^-18 of themselves: one would round as coarsely as the result, three (all of
    // their bits) take 667 us for 571 (1,024 x 11 x 363 heads forward and backward).  The error against 64 bits is the same in
    // its first digits, the result's own rounding (0.0017 of the root mean square); about one result in 3,000 is rounded the
    // other way than one of fp32 products
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool some = HALVES == 2 || e == 0;
      const float p0 = some ? P[HALVES == 2 ? e >> 1 : 0][2 * (e & 1)] : 0.0f, p1 = some ? P[HALVES == 2 ? e >> 1 : 0][2 * (e & 1) + 1] : 0.0f;
      hi[e] = pack(p0, p1);
      lo[e] = pack(p0 - low(hi[e]), p1 - high(hi[e]));
    }
#pragma unroll
    for (int q = 0; q < P_::kWords; ++q) {
      float O[4] = {};
      const uint32_t b0 = transpose(c.r[0][q]), b1 = HALVES == 2 ? transpose(c.r[kLast][q]) : 0u;
      mma_bf16(O, lo, b0, b1);
      mma_bf16(O, hi, b0, b1);
      out.r[0][q] = keep0 ? pack(O[0], O[1]) : 0u;
      if (HALVES == 2) out.r[kLast][q] = keep1 ? pack(O[2], O[3]) : 0u;
    }
  }
  return out;
}

// Blocks per SM that the registers are cut for (0: the compiler's choice): bf16 backwards 343 us with 4, 365 with its 3; forwards its 6
// take 180 us and a cut to the same 6 takes 190
template <typename T, int DP, bool BWD>
constexpr int kShortBlocks = BWD && sizeof(T) == 2 && DP <= 32 ? 4 : 0;

template <typename T, int DP, bool BWD, int HALVES>
__global__ void __launch_bounds__(kThreads, kShortBlocks<T, DP, BWD>) short_kernel(const __grid_constant__ Short p) {
  const uint32_t first = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), stride = gridDim.x * (kThreads / 32);
  uint32_t b = first / p.H, h = first - b * p.H;
  Piece<T, DP, HALVES> q, k, v, go;
  int rows = 0;
  auto load = [&] {
    rows = length_of(p.lengths, p.length_bytes, b, p.T);
    auto at = [&](const Rows& r) { return static_cast<const T*>(r.at) + b * r.b + h * r.h; };
    q.load(at(p.q), p.q.t, rows, p.dim_k);
    k.load(at(p.k), p.k.t, rows, p.dim_k);
    v.load(at(p.v), p.v.t, rows, p.dim_v);
    if constexpr (BWD) go.load(at(p.go), p.go.t, rows, p.dim_v);
  };
  if (first < p.items) load();
  for (uint32_t at = first; at < p.items;) {
    const Piece<T, DP, HALVES> q0 = q, k0 = k, v0 = v, go0 = go;
    const uint32_t b0 = b, h0 = h;
    const int rows0 = rows;
    const float log2_a = log2_decay(p.log_decay, h);
    // the next item's rows are on their way while this one's are used
    b += p.step_b, h += p.step_h;
    if (h >= static_cast<uint32_t>(p.H)) h -= p.H, ++b;
    at += stride;                                  // below 2^31: B H is below 2^30
    if (at < p.items) load();
    const int64_t row = (static_cast<int64_t>(b0) * p.T * p.H + h0);
    const int64_t sk = static_cast<int64_t>(p.H) * p.dim_k, sv = static_cast<int64_t>(p.H) * p.dim_v;
    const PairWeights forward(log2_a, false, p.scale);
    if constexpr (!BWD) {
      attend<T, DP, HALVES>(q0, k0, v0, forward, false, rows0).store(static_cast<T*>(p.o) + row * p.dim_v, sv, p.T, p.dim_v);
    } else {
      attend<T, DP, HALVES>(go0, v0, k0, forward, false, rows0).store(static_cast<T*>(p.dq) + row * p.dim_k, sk, p.T, p.dim_k);
      const PairWeights back(log2_a, true, p.scale);
      attend<T, DP, HALVES>(v0, go0, q0, back, true, rows0).store(static_cast<T*>(p.dk) + row * p.dim_k, sk, p.T, p.dim_k);
      attend<T, DP, HALVES>(k0, q0, go0, back, true, rows0).store(static_cast<T*>(p.dv) + row * p.dim_v, sv, p.T, p.dim_v);
    }
  }
}

// ---- one position --------------------------------------------------------------------------------------------------
// The state updated and read once: memory alone bounds it (64 x 676 heads of 32 x 32: 354 MB in 64 us, 5.7 TB/s; a block per head
// and a thread per column took 178).  WARPS warps per sequence and head, each some rows of the state; LV
// lanes of four columns across a row, so that a lane has 16-byte pieces of kUnroll rows under way.
struct Step {
  const void *q, *k, *v;
  void* o;
  const float *log_decay, *state;
  float* new_state;
  uint32_t items;               // B H
  int H, dk, dv;
  int64_t qb, qh, kb, kh, vb, vh;
  float scale;
};

template <typename T, int LV, int WARPS>
__global__ void __launch_bounds__(kThreads) step_kernel(const __grid_constant__ Step p) {
  constexpr int kUnroll = 8, kAcross = 32 / LV;      // rows at a time
  __shared__ float4 sums[WARPS > 1 ? kThreads : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WARPS;
  const uint32_t at = blockIdx.x * (kThreads / 32 / WARPS) + warp / WARPS;
  const bool there = at < p.items;
  const uint32_t b = there ? at / p.H : 0;
  const int h = there ? static_cast<int>(at - b * p.H) : 0;
  const int col = lane % LV * 4, share = (p.dk + WARPS - 1) / WARPS;
  const int row0 = part * share + lane / LV, end = min(p.dk, (part + 1) * share);
  const bool has = there && col < p.dv;
  const T* q = static_cast<const T*>(p.q) + b * p.qb + h * p.qh;
  const T* k = static_cast<const T*>(p.k) + b * p.kb + h * p.kh;
  const T* v = static_cast<const T*>(p.v) + b * p.vb + h * p.vh + col;
  const float a = expf(p.log_decay[h]);
  float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o = c;
  if (has) c = make_float4(load_f32(v), load_f32(v + 1), load_f32(v + 2), load_f32(v + 3));
  const int64_t base = static_cast<int64_t>(at) * p.dk * p.dv + col;
  for (int r0 = row0; r0 - lane / LV < end; r0 += kUnroll * kAcross) {
    float4 s[kUnroll];
    float kr[kUnroll], qr[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int row = r0 + u * kAcross;
      if (has && row < end) {
        s[u] = *reinterpret_cast<const float4*>(p.state + base + row * p.dv);
        kr[u] = load_f32(k + row), qr[u] = load_f32(q + row);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int row = r0 + u * kAcross;
      if (has && row < end) {
        s[u].x = fmaf(kr[u], c.x, a * s[u].x), s[u].y = fmaf(kr[u], c.y, a * s[u].y);
        s[u].z = fmaf(kr[u], c.z, a * s[u].z), s[u].w = fmaf(kr[u], c.w, a * s[u].w);
        *reinterpret_cast<float4*>(p.new_state + base + row * p.dv) = s[u];
        o.x = fmaf(qr[u], s[u].x, o.x), o.y = fmaf(qr[u], s[u].y, o.y);
        o.z = fmaf(qr[u], s[u].z, o.z), o.w = fmaf(qr[u], s[u].w, o.w);
      }
    }
  }
#pragma unroll
  for (int m = LV; m < 32; m *= 2) {
    o.x += __shfl_xor_sync(0xffffffffu, o.x, m), o.y += __shfl_xor_sync(0xffffffffu, o.y, m);
    o.z += __shfl_xor_sync(0xffffffffu, o.z, m), o.w += __shfl_xor_sync(0xffffffffu, o.w, m);
  }
  if constexpr (WARPS > 1) {
    sums[threadIdx.x] = o;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int w = 1; w < WARPS; ++w) {
        const float4 t = sums[threadIdx.x + 32 * w];
        o.x += t.x, o.y += t.y, o.z += t.z, o.w += t.w;
      }
    }
  }
  if (has && part == 0 && lane < LV) {
    T* out = static_cast<T*>(p.o) + static_cast<int64_t>(at) * p.dv + col;
    store_f32(out, p.scale * o.x), store_f32(out + 1, p.scale * o.y), store_f32(out + 2, p.scale * o.z), store_f32(out + 3, p.scale * o.w);
  }
}

// The same for states whose rows are no whole 16-byte pieces: a block per sequence and head, a thread per column
template <typename T>
__global__ void __launch_bounds__(kThreads) step_columns_kernel(const __grid_constant__ Step p) {
  const uint32_t at = blockIdx.x, b = at / p.H;
  const int h = static_cast<int>(at - b * p.H), j = threadIdx.x;
  if (j >= p.dv) return;
  const T* q = static_cast<const T*>(p.q) + b * p.qb + h * p.qh;
  const T* k = static_cast<const T*>(p.k) + b * p.kb + h * p.kh;
  const float a = expf(p.log_decay[h]), c = load_f32(static_cast<const T*>(p.v) + b * p.vb + h * p.vh + j);
  float sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < p.dk; ++i) {
    const int64_t e = (static_cast<int64_t>(at) * p.dk + i) * p.dv + j;
    const float s = fmaf(load_f32(k + i), c, a * p.state[e]);
    p.new_state[e] = s;
    sum = fmaf(load_f32(q + i), s, sum);
  }
  store_f32(static_cast<T*>(p.o) + static_cast<int64_t>(at) * p.dv + j, p.scale * sum);
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail(BPC_ERR_LAUNCH, std::string(what) + " launch: " + cudaGetErrorString(e));
}

int size_of(int32_t dtype) { return dtype == BPC_DTYPE_F32 ? 4 : dtype == BPC_DTYPE_BF16 ? 2 : 0; }

bool aligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// f(the padded head size as a type's value)
template <typename F>
auto with_dim(int dim, F f) {
  if (dim <= 16) return f(std::integral_constant<int, 16>());
  if (dim <= 32) return f(std::integral_constant<int, 32>());
  if (dim <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}
template <typename T>
struct Type {
  typedef T type;
};
template <typename F>
auto with_type(int32_t dtype, F f) {
  if (dtype == BPC_DTYPE_F32) return f(Type<float>());
  return f(Type<__nv_bfloat16>());
}

// Groups of scan_kernel's warps that are resident
int64_t resident_groups(int dim, int size) {
  return static_cast<int64_t>(num_sms()) * with_dim(dim, [&](auto d) {
    constexpr int DP = decltype(d)::value;
    return size == 4 ? Tile<float, DP>::kBlocks * Tile<float, DP>::kGroups : Tile<__nv_bfloat16, DP>::kBlocks * Tile<__nv_bfloat16, DP>::kGroups;
  });
}

template <typename T, int DP, bool REV, bool OUT, int SPLIT>
int launch_scan(const Scan& p, const Scan* second, bool follows, cudaStream_t s) {
  using L = Tile<T, DP>;
  const void* fn = reinterpret_cast<const void*>(&scan_kernel<T, DP, REV, OUT, SPLIT>);
  if (int e = allow_smem(fn, L::kSmem)) return e;
  Scans all{{p, second ? *second : p}, p.items, second ? 2 * p.items : p.items};
  const unsigned grid = std::min<unsigned>((all.total + L::kGroups - 1) / L::kGroups, L::kBlocks * num_sms());
  if (follows) {
    void* args[] = {&all};
    return launch_pdl(fn, dim3(grid), dim3(L::kThreads), L::kSmem, s, args, 1, "linear_attention");
  }
  scan_kernel<T, DP, REV, OUT, SPLIT><<<grid, L::kThreads, L::kSmem, s>>>(all);
  return launched("linear_attention");
}

// Into how many segments a sequence is cut: one where the heads alone keep the GPU busy, else as many as fill it once, of three
// chunks at least: the states' pass before costs a third of a chunk's time each and two launches
int segments_of(int64_t BH, int64_t T, int dim, int size) {
  return static_cast<int>(std::max<int64_t>(1, std::min(resident_groups(dim, size) / std::max<int64_t>(1, BH), T / (3 * kChunk))));
}

int64_t parts_bytes(int64_t BH, int64_t T, int da, int dc, int size) {
  return BH * (segments_of(BH, T, std::max(da, dc), size) - 1) * da * dc * static_cast<int64_t>(sizeof(float));
}

// A scan, and `second` (or null) beside it: the one with b and c exchanged, which starts from the same states the other way
// round.  turned_parts: the segments' states of such a scan that has run before, or null.
template <bool REV>
int run_scan(Scan p, Scan* second, int64_t B, int32_t dtype, float* workspace, const float* turned_parts, cudaStream_t s) {
  const int dim = std::max(p.da, p.dc);
  const int64_t BH = B * p.H;
  const int want = segments_of(BH, p.T, dim, size_of(dtype));
  p.segment = std::max(kChunk, ((p.T + want - 1) / want + kChunk - 1) / kChunk * kChunk);
  p.segments = std::max(1, (p.T + p.segment - 1) / p.segment);
  p.items = static_cast<uint32_t>(BH * p.segments);
  p.parts = workspace;
  if (turned_parts) p.parts = const_cast<float*>(turned_parts), p.parts_t = true;
  if (second) {
    second->segment = p.segment, second->segments = p.segments, second->items = p.items, second->parts = p.parts;
    second->parts_t = true;
  }
  return with_type(dtype, [&](auto type) {
    return with_dim(dim, [&](auto d) {
      typedef typename decltype(type)::type T;
      constexpr int DP = decltype(d)::value;
      // the state handed out is fp32: it needs every bit of the weighted rows; a bf16 result alone does with 16
      constexpr int kFew = sizeof(T) == 4 ? 3 : 2;
      const bool parts = p.segments > 1 && !turned_parts;
      if (parts) {
        if (int e = p.last ? launch_scan<T, DP, REV, false, 3>(p, nullptr, false, s) : launch_scan<T, DP, REV, false, kFew>(p, nullptr, false, s))
          return e;
        int per = (p.da * p.dc + 255) / 256;
        void* args[] = {&p, &per};
        if (int e = launch_pdl(reinterpret_cast<const void*>(&join_kernel<REV>), dim3(static_cast<unsigned>(BH * per)), dim3(256), 0, s, args, 1,
                               "linear_attention"))
          return e;
      }
      return p.last ? launch_scan<T, DP, REV, true, 3>(p, second, parts, s) : launch_scan<T, DP, REV, true, kFew>(p, second, parts, s);
    });
  });
}

template <typename T, int DP, bool BWD, int HALVES>
int launch_short(Short p, cudaStream_t s) {
  int blocks = 0;
  if (int e = resident_blocks(reinterpret_cast<const void*>(&short_kernel<T, DP, BWD, HALVES>), kThreads, "linear_attention", &blocks))
    return e;
  const uint32_t warps = kThreads / 32;
  const unsigned grid = std::min<unsigned>((p.items + warps - 1) / warps, blocks * num_sms());
  p.step_b = grid * warps / p.H, p.step_h = grid * warps % p.H;
  short_kernel<T, DP, BWD, HALVES><<<grid, kThreads, 0, s>>>(p);
  return launched("linear_attention");
}

template <bool BWD, int HALVES>
int run_short_of(const Short& p, int32_t dtype, cudaStream_t s) {
  return with_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    const int dim = std::max(p.dim_k, p.dim_v);
    if (dim <= 16) return launch_short<T, 16, BWD, HALVES>(p, s);
    if constexpr (sizeof(T) == 2)
      if (dim > 32) return launch_short<T, 64, BWD, HALVES>(p, s);
    return launch_short<T, 32, BWD, HALVES>(p, s);
  });
}

template <bool BWD>
int run_short(const Short& p, int32_t dtype, cudaStream_t s) {
  return p.T <= 8 ? run_short_of<BWD, 1>(p, dtype, s) : run_short_of<BWD, 2>(p, dtype, s);
}

// Head sizes that short_kernel holds in registers
int short_dim(int size) { return size == 4 ? 32 : 64; }

// 16-byte copies need rows of whole 16-byte pieces on 16-byte boundaries
bool copies_whole(const Rows& r, int dim, int size) {
  return aligned(r.at, 16) && dim * size % 16 == 0 && r.b * size % 16 == 0 && r.t * size % 16 == 0 && r.h * size % 16 == 0;
}

Scan make_scan(const Rows& a, const Rows& b, const Rows& c, void* out, const float* log_decay, const float* first, bool first_t,
               float* last, const void* lengths, int length_bytes, int64_t T, int H, int da, int dc, float in, float scale, int size) {
  Scan p = {};
  p.a = a, p.b = b, p.c = c;
  p.out = out;
  p.log_decay = log_decay;
  p.first = first, p.first_t = first_t, p.last = last;
  p.lengths = lengths, p.length_bytes = length_bytes;
  p.T = static_cast<int>(T), p.H = H, p.da = da, p.dc = dc;
  p.in_scale = in, p.out_scale = scale;
  p.vec = T > 0 && copies_whole(a, da, size) && copies_whole(b, da, size) && copies_whole(c, dc, size);
  p.out_vec = aligned(out, 16) && dc * size % (size == 4 ? 8 : 16) == 0;
  return p;
}

int check_common(const std::string& what, int64_t B, int64_t T, int32_t H, int32_t dk, int32_t dv, const void* lengths,
                 int32_t length_bytes, const int64_t* strides, int n_strides, float scale, int32_t dtype,
                 const float* log_decay) {
  auto bad = [&](const char* m) { return fail(BPC_ERR_ARG, what + ": " + m); };
  if (B < 0 || T < 0 || H < 0 || T > (1 << 30)) return bad("batch, length and heads must not be negative, length <= 2^30");
  if (H && B > 0x3fffffff / H) return bad("batch x heads must be below 2^30");      // items of two scans are counted in 32 bits
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

// Whether two states of `count` values share memory
bool overlap(const void* a, const void* b, int64_t count) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a), to = reinterpret_cast<uintptr_t>(b), bytes = sizeof(float) * static_cast<uintptr_t>(count);
  return a && b && at < to + bytes && to < at + bytes;
}

Rows rows_of(const void* p, const int64_t* s) { return {p, s[0], s[1], s[2]}; }

}  // namespace

}  // namespace bpc

using namespace bpc;

extern "C" size_t bpc_linear_attention_workspace_size(int64_t B, int64_t T, int32_t H, int32_t dk, int32_t dv,
                                                      int32_t dtype, int32_t backward) {
  if (B < 1 || T < 0 || H < 1 || dk < 1 || dk > kMaxDim || dv < 1 || dv > kMaxDim || !size_of(dtype)) return 0;
  return static_cast<size_t>(std::max<int64_t>(16, parts_bytes(B * H, T, dk, dv, size_of(dtype))));
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
  // a block may write a sequence's last state before another has read its first
  if (overlap(state, new_state, B * H * dk * dv)) return fail(BPC_ERR_ARG, "linear_attention: new_state overlaps state");
  if (workspace_bytes < bpc_linear_attention_workspace_size(B, T, H, dk, dv, dtype, 0))
    return fail(BPC_ERR_SPACE, "linear_attention: workspace too small");
  const Rows rq = rows_of(q, strides), rk = rows_of(k, strides + 3), rv = rows_of(v, strides + 6);
  // In registers where there is no state to carry.  1,024 x 11 x 363 bf16 heads of 32 take 184 us, and chunk by chunk 1,340 with a
  // last state and 1,996 with a first one, whose 1.5 GB alone are 236 at the copy's rate; 16 positions x 256 heads 170, 952 and 1,418
  if (T && T <= kShort && !state && !new_state && std::max(dk, dv) <= short_dim(size) && copies_whole(rq, dk, size) &&
      copies_whole(rk, dk, size) && copies_whole(rv, dv, size) && aligned(o, 16)) {
    const Short p{rq, rk, rv, {}, o, nullptr, nullptr, nullptr, log_decay, lengths, length_bytes, static_cast<int>(T), H, dk, dv,
                  scale, static_cast<uint32_t>(B * H), 0, 0};
    return run_short<false>(p, dtype, reinterpret_cast<cudaStream_t>(stream));
  }
  const Scan p = make_scan(rq, rk, rv, o, log_decay, state, false,
                           new_state, lengths, length_bytes, T, H, dk, dv, 1.0f, scale, size);
  return run_scan<false>(p, nullptr, B, dtype, static_cast<float*>(workspace), nullptr, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int bpc_linear_attention_bwd(const void* q, const void* k, const void* v, const void* go, const float* log_decay,
                                        const float* state, const float* grad_state, const void* fwd_workspace,
                                        const void* lengths, int32_t length_bytes, void* dq, void* dk_out, void* dv_out, float* dstate, int64_t B,
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
  if (!aligned(state, 16) || !aligned(grad_state, 16) || !aligned(dstate, 16) || !aligned(workspace, 16) || !aligned(fwd_workspace, 16))
    return fail(BPC_ERR_ARG, "linear_attention backward: buffer not aligned to its type (states and workspace: 16 bytes)");
  if (overlap(grad_state, dstate, B * H * dk * dv) || overlap(state, dstate, B * H * dk * dv))
    return fail(BPC_ERR_ARG, "linear_attention backward: dstate overlaps state or grad_state");
  if (workspace_bytes < bpc_linear_attention_workspace_size(B, T, H, dk, dv, dtype, 1))
    return fail(BPC_ERR_SPACE, "linear_attention backward: workspace too small");
  const Rows rq = rows_of(q, strides), rk = rows_of(k, strides + 3), rv = rows_of(v, strides + 6), rg = rows_of(go, strides + 9);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (T && T <= kShort && !state && !grad_state && !dstate && std::max(dk, dv) <= short_dim(size) && copies_whole(rq, dk, size) &&
      copies_whole(rk, dk, size) && copies_whole(rv, dv, size) && copies_whole(rg, dv, size) && aligned(dq, 16) &&
      aligned(dk_out, 16) && aligned(dv_out, 16)) {
    const Short p{rq, rk, rv, rg, nullptr, dq, dk_out, dv_out, log_decay, lengths, length_bytes, static_cast<int>(T), H, dk, dv,
                  scale, static_cast<uint32_t>(B * H), 0, 0};
    return run_short<true>(p, dtype, s);
  }
  float* ws = static_cast<float*>(workspace);
  if (T) {
    const Scan pq = make_scan(rg, rv, rk, dq, log_decay, state, true, nullptr, lengths, length_bytes, T, H, dv, dk, 1.0f, scale, size);
    if (int e = run_scan<false>(pq, nullptr, B, dtype, ws, static_cast<const float*>(fwd_workspace), s)) return e;
  }
  const Scan pv = make_scan(rk, rq, rg, dv_out, log_decay, grad_state, false, dstate, lengths, length_bytes, T, H, dk, dv, scale, 1.0f, size);
  if (!T) return run_scan<true>(pv, nullptr, B, dtype, ws, nullptr, s);
  Scan pk = make_scan(rv, rg, rq, dk_out, log_decay, grad_state, true, nullptr, lengths, length_bytes, T, H, dv, dk, scale, 1.0f, size);
  return run_scan<true>(pv, &pk, B, dtype, ws, nullptr, s);
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
  if (state != new_state && overlap(state, new_state, B * H * dk * dv))
    return fail(BPC_ERR_ARG, "linear_attention_step: new_state overlaps state (give the same buffer to update it in place)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Step p{q, k, v, o, log_decay, state, new_state, static_cast<uint32_t>(B * H), H, dk, dv,
               strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], scale};
  with_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    if (dv % 4 || !aligned(state, 16) || !aligned(new_state, 16)) {
      step_columns_kernel<T><<<p.items, kThreads, 0, s>>>(p);
      return 0;
    }
    // states of more than 4 KB by four warps: 64 x 64 and 128 x 128 have as much under way per state as 32 x 32
    auto run = [&](auto lanes) {
      constexpr int LV = decltype(lanes)::value;
      if (dk * dv > 1024) step_kernel<T, LV, 4><<<p.items, kThreads, 0, s>>>(p);
      else step_kernel<T, LV, 1><<<(p.items + 3) / 4, kThreads, 0, s>>>(p);
    };
    if (dv <= 16) run(std::integral_constant<int, 4>());
    else if (dv <= 32) run(std::integral_constant<int, 8>());
    else if (dv <= 64) run(std::integral_constant<int, 16>());
    else run(std::integral_constant<int, 32>());
    return 0;
  });
  return launched(what);
}
