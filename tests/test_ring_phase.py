"""The ring of the few-token embedding gradient after a wait that ran out, on a model of its barriers: what is still being
copied into a slot is waited for, however many uses had been issued.  Runs without a GPU (the header is plain C++)."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "codecoder_b200", "csrc")

MODEL = r"""
#include <cstdio>
#include "ring_phase.h"
// a barrier with `done` whole phases lets a wait for parity p through iff the phase under way has the other parity
static bool passes(int done, unsigned p) { return (done & 1u) != p; }
int main() {
  for (int stages = 1; stages <= 5; ++stages)
    for (int issued = 1; issued <= 4 * stages + 3; ++issued)
      for (int slot = 0; slot < stages && slot < issued; ++slot) {
        int uses = 0, last = -1;
        for (int k = slot; k < issued; k += stages) ++uses, last = k;
        if (bpc::ring_last_use(issued, slot, stages) != last) return std::printf("last use\n"), 1;
        const unsigned p = bpc::ring_parity(last, stages);
        // every use but the last is complete (its slot was taken again); the last may be or not
        if (passes(uses - 1, p) || !passes(uses, p)) return std::printf("wait %d %d %d\n", stages, issued, slot), 1;
      }
  return 0;
}
"""


def test_the_drain_waits_for_the_copies_under_way(tmp_path):
    (tmp_path / "model.cpp").write_text(MODEL)
    exe = str(tmp_path / "model")
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(tmp_path / "model.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_the_kernel_drains_what_it_issued():
    src = open(os.path.join(CSRC, "embedding.cu")).read()
    drain = src[src.index("after a wait that ran out"):]
    drain = drain[:drain.index("__syncthreads")]
    assert "ring_last_use(issued, q, kFewStages)" in drain and not re.search(r"\bcopied\b", drain)


def test_a_warp_leaves_its_loop_as_a_whole():
    """The kernel's waits: a vote decides for the warp (at once, or on the outcome kept until the end of the stage), or no
    lane acts on the outcome."""
    src = open(os.path.join(CSRC, "embedding.cu")).read()
    waits = [m.start() for m in re.finditer(r"\bmbar_wait\(", src)]
    assert len(waits) >= 3
    for at in waits:
        line = src[src.rindex("\n", 0, at) + 1:at]
        kept = line.strip() == "const bool ok =" and len(re.findall(r"\bok\b", src[at:])) == 1 and \
            "if (!__all_sync(0xffffffffu, ok)) break;" in src[at:]
        assert line.endswith("__all_sync(0xffffffffu, ") or not line.strip() or kept, src[at - 80:at + 40]
