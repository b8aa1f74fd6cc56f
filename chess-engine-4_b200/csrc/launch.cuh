// Launch helpers shared by the kernels that start under their predecessor's tail.
#pragma once

#include <cuda_runtime.h>

#include <mutex>
#include <set>
#include <utility>

#include "internal.h"

namespace ce4b {

// Opt each kernel instantiation into the dynamic shared memory it needs, once per device.
template <class K>
void ensure_smem(K kernel, int bytes) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  const auto key = std::make_pair(dev, reinterpret_cast<const void*>(kernel));
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(key)) return;
  check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
             "cudaFuncSetAttribute(max dynamic smem)");
  done.insert(key);
}

template <class K, class... Args>
void launch(K kernel, dim3 grid, int threads, int smem, int cluster_x, cudaStream_t s,
            Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  // Every kernel launched here waits for its predecessor (grid_dependency_wait) before touching
  // global memory, so it may be launched programmatically: its CTAs take SMs as the
  // previous kernel's CTAs leave and run their prologue under that kernel's tail.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  unsigned n_attr = 1;
  if (cluster_x > 0) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster_x);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    n_attr = 2;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n_attr;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), "kernel launch");
}

}  // namespace ce4b
