// What the host sides of the operators share (abi.cu, kv4.cu): errors, the head of a workspace, launches,
// and the scheduling decision of the prefill kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/msgl_b200.h"

namespace msgl_host {

// Keeps the message for msgl_last_error_string and returns the code.
int fail(int code, const std::string& msg);
int cuda_fail(const char* op, cudaError_t e);

// Head of every workspace: the device status word (first 256 bytes), then kTicketSlots arrival
// counters of split-KV pieces at a fixed place, so that a buffer re-used by calls of different
// shapes never finds anything but the zeros the kernels leave there.
constexpr size_t kTicketSlots = 16384;
constexpr size_t kStatusBytes = 256 + kTicketSlots * sizeof(int);

inline bool aligned16(const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; }

// SMs of the current device, <0 on error.
int sm_count_cached();

// Dynamic shared memory of a kernel, set once per kernel, device and thread (the runtime call takes
// longer than the rest of a launch's preparation).
template <typename K>
cudaError_t allow_smem(K kernel, int bytes) {
  struct Done {
    const void* fn;
    int dev, bytes;
  };
  static thread_local Done done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const void* fn = reinterpret_cast<const void*>(kernel);
  Done& d = done[((reinterpret_cast<uintptr_t>(fn) >> 4) ^ dev) % 64];
  if (d.fn == fn && d.dev == dev && d.bytes == bytes) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) d = Done{fn, dev, bytes};
  return e;
}

// Launches `kernel` so that its CTAs may be scheduled while the previous kernel of the
// stream drains (programmatic dependent launch); the kernel itself waits for the previous
// kernel's memory with griddepcontrol.wait before it touches global memory.
template <typename... P, typename... A>
cudaError_t launch_clusters(int cluster, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                            const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                             const A&... args) {
  return launch_clusters(1, kernel, grid, block, smem, s, args...);
}

// Tensor maps over a pool, see make_pool_map.
enum class PoolBox {
  kPage,   // 2-D, 16 token rows x 64 elements (128 bytes) of one head
  kRow,    // 2-D, one row of those, for tile::gather4
  kHead,   // 3-D (64 elements, slots, blocks of 64 elements of a row): 16 token rows x all head_dim elements of one head, a block
           // of columns after the other, as the decode kernel's tiles lie in shared memory.  (A copy instruction costs
           // its warp 67 cycles whatever its size: one per tile instead of two or four.)
  kPacked, // 2-D, for tile::gather4: a pool held in 4 bits as rows of 1152 bytes (144 elements of 8), one or two to a block of a head
};
bool make_pool_map(CUtensorMap* out, PoolBox form, const void* base, int64_t num_slots, int num_kv_heads, int head_dim,
                   int dtype);
// Tensor map over the query rows for tile::gather4.
bool make_query_row_map(CUtensorMap* out, const void* q, int total_q, int num_q_heads, int head_dim, int dtype);
// Tensor map over the query tensor whose box is the 128 packed rows of a query sub-tile; false where
// the group does not divide 128.
bool make_query_tensor_map(CUtensorMap* out, const void* q, int total_q, int num_q_heads, int group,
                           int head_dim, int dtype);

// ---- prefill scheduling decision (shared by the workspace query and the launch)
struct PrefillPlan {
  int kv_chunk;        // 0 = no kv split
  int64_t items;       // grid.x
  size_t part_o_bytes, part_ml_bytes, plan_bytes;
  bool fused_merge;    // the CTA that arrives last at a unit merges it (else: a second launch)
};
bool prefill_pairs(int batch, int total_q, int64_t total_kv, int group, int num_kv_heads, int head_dim,
                   int max_len_extend, bool cross, int window, int kv_chunk, bool paged, int sms);
bool prefill_short_q(int max_len_extend, int group, int head_dim);
PrefillPlan plan_prefill(int batch, int total_q, int64_t total_kv, int hq, int hkv, int head_dim,
                         int max_len_extend, int window, int sms);

}  // namespace msgl_host
