"""A refused launch or attribute leaves no error behind for the next kernel's check, which reads the thread's last one.  On a
runtime that refuses what it is told to, without a GPU."""
import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "codecoder_b200", "csrc")

RUNTIME = r"""
#include <cstdio>
#include "bpc_internal.h"
static cudaError_t last = cudaSuccess;
static bool refuse = true;
static int attributes = 0, launches = 0;
static cudaError_t answer(cudaError_t e) { return refuse ? last = e : cudaSuccess; }
extern "C" {
cudaError_t cudaGetLastError() { const cudaError_t e = last; last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t) { return "refused"; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { ++attributes; return answer(cudaErrorInvalidValue); }
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessor(int*, const void*, int, size_t) { return answer(cudaErrorInvalidValue); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { ++launches; return answer(cudaErrorInvalidConfiguration); }
}
namespace bpc {
static std::string message;
int fail(int code, const std::string& m) { message = m; return code; }
}
using namespace bpc;
int main() {
  int kernel = 0;
  const int codes[] = {allow_smem(&kernel, 300000), launch_pdl(&kernel, dim3(1), dim3(32), 0, nullptr, nullptr, 2, "this"),
                       launch_clusters(&kernel, dim3(1), dim3(32), 0, nullptr, nullptr, 2, "that"),
                       launch_clusters(&kernel, dim3(1), dim3(32), 100000, nullptr, nullptr, 1, "that")};
  for (int code : codes)
    if (code != BPC_ERR_LAUNCH) return std::printf("code %d\n", code), 1;
  if (message != "cudaFuncSetAttribute: refused" || last != cudaSuccess) return std::printf("left behind: %d\n", last), 1;
  if (attributes != 2 || launches != 2) return std::printf("calls %d %d\n", attributes, launches), 1;
  launch_pdl(&kernel, dim3(1), dim3(32), 0, nullptr, nullptr, 1, "this");
  if (message != "this launch: refused" || last != cudaSuccess) return std::printf("left behind: %d\n", last), 1;
  int blocks = 0;
  if (resident_blocks(&kernel, 128, "these", &blocks) != BPC_ERR_LAUNCH || message != "these occupancy: refused" || last != cudaSuccess)
    return std::printf("left behind: %d\n", last), 1;
  refuse = false;               // what was refused is not remembered as granted
  if (allow_smem(&kernel, 100000) || attributes != 3 || allow_smem(&kernel, 50000) || attributes != 3) return std::printf("granted\n"), 1;
  return launch_clusters(&kernel, dim3(1), dim3(32), 100000, nullptr, nullptr, 4, "that");
}
"""


def test_a_refusal_leaves_no_error_behind(tmp_path):
    from codecoder_b200.build import nvcc
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    (tmp_path / "runtime.cpp").write_text(RUNTIME)
    exe = str(tmp_path / "launch")
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", f"-I{os.path.join(REPO, 'include')}", f"-isystem{cuda}", "-x", "c++",
                    os.path.join(CSRC, "launch.cu"), str(tmp_path / "runtime.cpp"), "-o", exe, "-lpthread"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
