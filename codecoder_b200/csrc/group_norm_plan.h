// How the group normalisation cuts its features into pieces of work: plain C++, shared by the kernels and the host.
#pragma once
#include <algorithm>
#include <cstdint>

namespace bpc {
namespace gn {

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
constexpr int kRows = 8;             // of a thread's registers
constexpr int kTileVec = 4;          // elements of a tile's access, whatever their type: eight rows of eight would not stay in registers
struct Plan {
  Kind kind;
  int vec;                        // elements per access
  int lanes, slots, rows;         // units
  int slab, slabs, V;             // tiles: channels of a slab, slabs, threads across one
  int chunks, chunk_rows;
  bool fused;
  int threads;
};

constexpr int kUnitThreads = 512;    // at most
constexpr int kTileThreads = 256;

// Dynamic shared memory of a block: one that a launch can have, and what a kernel takes.
constexpr int kBlockSmem = 227 * 1024;
// units: samples that are on their way or worked on, of which a thread copies so many bytes each: four, or three where the largest
// block has no room for four.  That is fp32 with fp32 gradients and four slots, 136 bytes: 278,528 or 208,896 for 512 threads.
// Smaller blocks of it lose nothing by the same depth (65,536 x 512 in one group forward and backward 152 us with four, 144 with
// three; 20,000 x 33 x 104 in 13 groups 408 and 366), and tiles would take 547 us for 4,096 x 8,192 in 16 groups: 156.
constexpr int units_depth(int thread_bytes) { return 4 * thread_bytes * kUnitThreads <= kBlockSmem ? 4 : 3; }
// a ring of them (single elements of 2 bytes are not copied), backwards with gy's and the statistics beside x's, and at the end a
// row of sums for each of the block's rows
constexpr int copied_bytes(int size, int vec) { return size * vec >= 4 ? size * vec : 0; }
constexpr int units_bytes(int x_copied, int y_copied, int slots, bool backward) { return backward ? (x_copied + y_copied) * slots + 8 : x_copied * slots; }
inline int units_smem(const Plan& p, const Shape& s, int size, int y_size, bool backward) {
  const int thread = units_bytes(copied_bytes(size, p.vec), copied_bytes(y_size, p.vec), p.slots, backward);
  const int ring = units_depth(thread) * thread * p.threads;
  return backward ? std::max(ring, p.rows * static_cast<int>(s.N) * s.C * static_cast<int>(sizeof(float))) : ring;
}

// Whole accesses are taken where the pointers and strides allow it (`aligned`) and the groups hold whole ones: of kTileVec
// elements in tiles, in units of `full`, SLOTS of them a lane: two where there are two forwards, as the joins and the addresses are
// half of the rest; one backwards, where the sums of gradients fill the registers, and of kTileVec where one is not enough.
inline Plan make_plan(const Shape& s, int size, int sms, bool aligned, bool backward) {
  Plan p = {};
  const int cg = s.C / s.G;
  int full = 16 / size;
  // small samples, of which a block per sample and slab would have little: 32-byte pieces of rows at least, or whole rows
  if (s.N * cg <= 128 * full && (s.N == 1 || cg * size >= 32)) {
    if (backward && s.N * cg > 32 * full) full = kTileVec;
    p.vec = aligned && cg % full == 0 ? full : 1;
    const int vectors = static_cast<int>(s.N) * (cg / p.vec);
    p.slots = vectors > 64 ? 4 : vectors > (backward ? 32 : 1) ? 2 : 1;
    p.lanes = 1;
    while (p.lanes * p.slots < vectors) p.lanes *= 2;
    if (p.lanes <= 32 && p.lanes * s.G <= kUnitThreads) {
      p.kind = kUnits;
      p.rows = std::max(1, 256 / (p.lanes * s.G));
      p.threads = (p.lanes * s.G * p.rows + 31) / 32 * 32;
      return p;
    }
  }
  p.vec = aligned && cg % kTileVec == 0 ? kTileVec : 1;
  const int across = cg / p.vec;
  if (across > kTileThreads) {
    p.kind = kWide;
    p.threads = 256;
    return p;
  }
  p.kind = kTiles;
  // slabs of 64-byte rows or one group, whichever is wider; of 32-byte rows where they keep the sample in a cluster
  for (int bytes = 64; bytes >= 32; bytes /= 2) {
    const int groups = std::min(s.G, std::max(1, std::min((bytes / size + cg - 1) / cg, kTileThreads / across)));
    p.slab = groups * cg;
    p.slabs = (s.G + groups - 1) / groups;
    p.V = p.slab / p.vec;
    const int lanes = kTileThreads / p.V;
    int64_t chunks = (s.N + static_cast<int64_t>(lanes) * kRows - 1) / (static_cast<int64_t>(lanes) * kRows);
    // few blocks: more chunks, down to two rows per thread
    while (chunks * 2 <= kCluster && s.B * p.slabs * chunks * 2 <= sms && s.N >= lanes * chunks * 4) chunks *= 2;
    p.fused = chunks <= kCluster;
    p.chunk_rows = static_cast<int>((s.N + chunks - 1) / chunks);
    p.chunks = static_cast<int>((s.N + p.chunk_rows - 1) / p.chunk_rows);
    p.threads = (std::min(lanes, p.chunk_rows) * p.V + 31) / 32 * 32;
    if (p.fused) break;
  }
  return p;
}

}  // namespace gn
}  // namespace bpc
