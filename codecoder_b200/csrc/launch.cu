// Kernel launches and their attributes on the host.  A call that is refused leaves no error behind: the next kernel's check reads
// the last one of its thread.  Plain C++ but for its name.
#include <atomic>
#include <map>
#include <mutex>
#include <string>
#include <utility>

#include "bpc_internal.h"

namespace bpc {

int refused(const std::string& what, cudaError_t e) {
  cudaGetLastError();
  return fail(BPC_ERR_LAUNCH, what + ": " + cudaGetErrorString(e));
}

int allow_smem(const void* fn, int bytes) {
  // the attribute is per device and kernel: remember the size set for each (device, kernel) pair and raise it when
  // a launch needs more
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> configured;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  auto it = configured.find({dev, fn});
  if (it != configured.end() && it->second >= bytes) return 0;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return refused("cudaFuncSetAttribute", e);
  configured[{dev, fn}] = bytes;
  return 0;
}

int launch_pdl(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, void** args, int cluster_x,
               const char* what) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = block;
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  if (cluster_x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster_x);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  lc.attrs = attr;
  lc.numAttrs = n;
  cudaError_t e = cudaLaunchKernelExC(&lc, fn, args);
  return e == cudaSuccess ? 0 : refused(std::string(what) + " launch", e);
}

int launch_clusters(const void* fn, dim3 grid, dim3 block, int smem, cudaStream_t stream, void** args, int cluster_x, const char* what) {
  if (smem > 32 * 1024)          // beside a few KB of static memory
    if (int e = allow_smem(fn, smem)) return e;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = block;
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster_x);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  lc.attrs = &attr;
  lc.numAttrs = cluster_x > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelExC(&lc, fn, args);
  return e == cudaSuccess ? 0 : refused(std::string(what) + " launch", e);
}

int resident_blocks(const void* fn, int threads, const char* what, int* blocks) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  int& n = known[{dev, fn}];
  if (n < 1) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, threads, 0);
    if (e != cudaSuccess || n < 1) {
      n = 0;
      return refused(std::string(what) + " occupancy", e);
    }
  }
  *blocks = n;
  return 0;
}

int num_sms() {
  static std::atomic<int> known{0};
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 1;
    known.store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace bpc
