"""How the group normalisation cuts its features: every launch that a plan asks for is one that a block can have.  Runs without
a GPU (the header is plain C++)."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "codecoder_b200", "csrc")

# Shared memory as a B200 gives it, and the kernels' own static part in `tiles` beside eight rows of x and of gy a thread.
SWEEP = r"""
#include <cstdio>
#include "group_norm_plan.h"
using namespace bpc::gn;
int main() {
  const int limit = 232448;
  long units = 0, narrowed = 0;
  for (int G = 1; G <= 513; ++G)
    for (int cg = 1; cg <= 1100; cg += cg < 72 ? 1 : cg < 512 ? 4 : 49)
      for (int N = 1; N <= 48 && N * cg <= 1100; ++N)
        for (int size : {2, 4})
          for (int y_size : {2, 4})
            for (bool aligned : {false, true})
              for (bool backward : {false, true}) {
                if (y_size > size) continue;
                const Shape s{5, N, G * cg, G, static_cast<int64_t>(N) * G * cg, G * cg, static_cast<int64_t>(N) * G * cg, G * cg};
                const Plan p = make_plan(s, size, 148, aligned, backward);
                if (p.threads < 32 || p.threads % 32 || p.threads > (p.kind == kUnits ? kUnitThreads : kTileThreads))
                  return std::printf("threads %d: %d groups of %d, %d rows\n", p.threads, G, cg, N), 1;
                if (p.kind != kUnits) continue;
                ++units;
                // counted here again: a stage of every vector that a thread copies, four deep or three
                int thread = size * p.vec >= 4 ? size * p.vec * p.slots : 0;
                if (backward) thread += (y_size * p.vec >= 4 ? y_size * p.vec * p.slots : 0) + 8;
                const int depth = 4 * thread * 512 <= limit ? 4 : 3;
                int bytes = depth * thread * p.threads;
                if (backward && bytes < p.rows * N * G * cg * 4) bytes = p.rows * N * G * cg * 4;
                if (units_smem(p, s, size, y_size, backward) != bytes)
                  return std::printf("bytes: %d groups of %d, %d rows\n", G, cg, N), 1;
                if (bytes > limit)
                  return std::printf("%d bytes: %d groups of %d, %d rows, sizes %d %d, backward %d\n", bytes, G, cg, N, size, y_size, backward), 1;
                // every vector of a group has a lane's slot, and every group its lanes
                if (p.lanes * p.slots * p.vec < N * cg || p.lanes > 32 || p.lanes * G * p.rows > p.threads)
                  return std::printf("lanes: %d groups of %d, %d rows\n", G, cg, N), 1;
                narrowed += backward && y_size < size && G >= 14;
              }
  return units < 100000 || narrowed == 0;
}
"""


def test_every_plan_can_be_launched(tmp_path):
    (tmp_path / "sweep.cpp").write_text(SWEEP)
    exe = str(tmp_path / "sweep")
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{CSRC}", str(tmp_path / "sweep.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
