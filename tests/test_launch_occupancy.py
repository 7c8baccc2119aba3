"""What the runtime answers about a kernel's occupancy is kept per device and kernel, whichever threads ask at once; a refusal is not
kept.  On a runtime of the test's own, without a GPU."""
import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "codecoder_b200", "csrc")

RUNTIME = r"""
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>
#include "bpc_internal.h"
static thread_local int device = 0;
static std::atomic<int> asked{0}, sms{0};
static bool refuse = false;
extern "C" {
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "refused"; }
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { ++sms; *v = 148; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void* fn, int threads, size_t) {
  ++asked;
  if (refuse) return cudaErrorInvalidValue;
  *n = device + *static_cast<const int*>(fn) * threads;       // this device's and this kernel's own
  return cudaSuccess;
}
}
namespace bpc {
int fail(int code, const std::string&) { return code; }
}
using namespace bpc;
int main() {
  static const int kernels[3] = {1, 2, 3};
  int n = 0;
  refuse = true;
  if (resident_blocks(&kernels[0], 128, "this", &n) != BPC_ERR_LAUNCH || asked != 1) return std::printf("refusal\n"), 1;
  refuse = false;
  std::atomic<int> wrong{0};
  std::vector<std::thread> threads;
  for (int t = 0; t < 16; ++t)
    threads.emplace_back([t, &wrong] {
      for (int k = 0; k < 20000; ++k) {
        device = (t + k) % 2;
        int n = 0;
        if (resident_blocks(&kernels[k % 3], 128, "this", &n) || n != device + kernels[k % 3] * 128 || num_sms() != 148) ++wrong;
      }
    });
  for (std::thread& t : threads) t.join();
  if (wrong || asked != 7) return std::printf("wrong %d, asked %d\n", wrong.load(), asked.load()), 1;
  return 0;
}
"""


def test_answers_are_kept_per_device_and_kernel(tmp_path):
    from codecoder_b200.build import nvcc
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    (tmp_path / "runtime.cpp").write_text(RUNTIME)
    exe = str(tmp_path / "occupancy")
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", f"-I{os.path.join(REPO, 'include')}",
                    f"-isystem{cuda}", "-x", "c++", os.path.join(CSRC, "launch.cu"), str(tmp_path / "runtime.cpp"), "-o", exe,
                    "-lpthread"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
