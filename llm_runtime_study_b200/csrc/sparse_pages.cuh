// Shared by sparse_pages.cu and sparse_attention.cu: the head size they are built for, and how a row of it lies on lanes.
#pragma once

#include <math_constants.h>

#include "common.cuh"

#ifndef HEAD_DIM
#error "HEAD_DIM must be given"
#endif

namespace b200 {

constexpr int kDim = HEAD_DIM;
static_assert(kDim % 16 == 0 && kDim >= 16 && kDim <= 256, "head sizes in steps of 16 up to 256");

// How a row of HEAD_DIM values is spread over lanes: 16-byte chunks, chunk i of lane l is l + i * lanes.
template <typename T> struct RowLanes {
  static constexpr int chunks = kDim * static_cast<int>(sizeof(T)) / 16;
  static constexpr int lanes = chunks % 8 == 0 ? 8 : (chunks % 4 == 0 ? 4 : 2);
  static constexpr int per_lane = chunks / lanes;
  static constexpr int values = per_lane * Vec<T>::n;      // channels a lane holds
};

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t in_cluster(uint32_t address, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(address), "r"(rank));
  return remote;
}
__device__ __forceinline__ float load_in_cluster(uint32_t address) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// The barrier alone, for CTAs that only stay until the others have read their shared memory.
__device__ __forceinline__ void cluster_leave() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
}

// As launch(), in clusters of `cluster` CTAs along x.
template <typename... Params, typename... Args>
inline void launch_clusters(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = cluster;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  const int first = pdl_enabled() ? 0 : 1;
  config.attrs = attributes + first;
  config.numAttrs = (cluster > 1 ? 2 : 1) - first;
  cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

}  // namespace b200
