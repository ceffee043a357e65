// What the host functions behind the C ABI share: error returns, the device handle, launch helpers.
#pragma once
#include "../../include/webgpt_b200.h"

#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <mutex>
#include <set>
#include <utility>

#define WGPT_EXPORT extern "C" __attribute__((visibility("default")))

// ------------------------------------------------------------------------------------------ errors
// Leaves the message for wgpt_last_error and returns the code.
int32_t fail(int32_t code, const char *fmt, ...);

#define CK(call)                                                                                   \
  do {                                                                                             \
    cudaError_t e__ = (call);                                                                      \
    if (e__ != cudaSuccess)                                                                        \
      return fail(e__ == cudaErrorMemoryAllocation ? WGPT_ERR_OOM : WGPT_ERR_CUDA, "%s: %s", #call, \
                  cudaGetErrorString(e__));                                                        \
  } while (0)

#define TRY(call)                 \
  do {                            \
    int32_t rc__ = (call);        \
    if (rc__ != WGPT_OK) return rc__; \
  } while (0)

#define REQUIRE(cond, code, ...) \
  do {                           \
    if (!(cond)) return fail((code), __VA_ARGS__); \
  } while (0)

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ------------------------------------------------------------------------------------------ device
constexpr int kJoinCounters = 4096;

struct wgpt_device {
  int ordinal;
  cudaStream_t stream;
  int precision;
  uint64_t launches;
  int sm_count;
  size_t smem_optin;
  void *scratch;  // library-owned workspace (split-K partial sums, temporaries of wgpt_attention)
  size_t scratch_cap;
  uint64_t scratch_gen;  // bumped whenever the workspace moves: recorded pass lists hold its old address
  int *d_err;     // device-side error word (out-of-range token id)
  float *tc_scratch;  // split-K partial tiles of the tensor-core GEMM (fixed size)
  size_t tc_scratch_bytes;
  bool pdl;       // launch the decode-chain kernels with programmatic dependent launch (WGPT_PDL=0 turns it off)
  bool graphs;    // replay decode steps as a CUDA graph (WGPT_GRAPH=0 turns it off)
  bool capturing;   // between wgpt_graph_begin and wgpt_graph_end
  uint64_t capture_launch0;
  bool block_gemv;  // layer GEMVs through gemv_block_kernel (WGPT_BLOCK_GEMV=0: register-streaming kernel)
  int deembed_tc_min_rows;   // fewest sequences whose de-embedding runs on the tensor-core GEMM (WGPT_DEEMBED_TC_ROWS)
  int gemv_stream_max_rows;  // most rows the register-streaming GEMV takes for a layer product (WGPT_GEMV_MAX_ROWS)
  unsigned int *d_work;  // two counters of gemv_loop_kernel (left zero by every launch)
  unsigned int *d_join;  // kJoinCounters counters of the paged attention's split groups (left zero by every launch)
  bool loop_gemv;     // products against matrices larger than L2 through gemv_loop_kernel (WGPT_LOOP_GEMV=0: off)
  int max_clusters[9];  // clusters of S CTAs of gemm_split_kernel resident at once with one CTA per SM
  bool fused_decode;  // single-sequence decode with two kernels per block (WGPT_FUSED_DECODE=0 turns it off)
};

#define LAUNCH(dev, kernel, grid, block, smem, ...)                       \
  do {                                                                    \
    kernel<<<(grid), (block), (smem), (dev)->stream>>>(__VA_ARGS__);      \
    (dev)->launches++;                                                    \
    CK(cudaGetLastError());                                               \
  } while (0)

// Lets a kernel take all the dynamic shared memory that its static part leaves, once per kernel and device. The limit is
// never lowered again: two threads that drive two devices handles share it, and one setting its own launch's size could
// undercut the other's between that one's setting and its launch.
static cudaError_t allow_smem_raw(const wgpt_device *dev, const void *kern, bool whole_carveout) {
  static std::mutex mu;
  static std::set<std::pair<const void *, int>> done;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kern, dev->ordinal})) return cudaSuccess;
  cudaFuncAttributes at;
  cudaError_t e = cudaFuncGetAttributes(&at, kern);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(dev->smem_optin - at.sharedSizeBytes));
  // the whole carveout, so that the next kernel's CTA fits on the SM beside this one's and fetches its weights early
  if (e == cudaSuccess && whole_carveout)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) done.insert({kern, dev->ordinal});
  return e;
}
template <typename K>
static cudaError_t allow_smem(const wgpt_device *dev, K kern, bool whole_carveout = false) {
  return allow_smem_raw(dev, reinterpret_cast<const void *>(kern), whole_carveout);
}

// Launch for kernels that call pdl_wait() before touching anything an earlier kernel wrote: with dev->pdl they
// carry the programmatic-serialisation attribute and may start while their predecessor is still running.
template <typename... KArgs, typename... Args>
static cudaError_t launch_ex(bool pdl, int cluster_z, cudaStream_t stream, void (*kernel)(KArgs...), dim3 grid,
                             dim3 block, size_t smem, Args... args);
// The same with clusters of cluster_x CTAs along x.
template <typename... KArgs, typename... Args>
static cudaError_t launch_ex_x(bool pdl, int cluster_x, cudaStream_t stream, void (*kernel)(KArgs...), dim3 grid,
                               dim3 block, size_t smem, const Args &...args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  attr[n].id = cudaLaunchAttributeClusterDimension;
  attr[n].val.clusterDim.x = (unsigned)cluster_x;
  attr[n].val.clusterDim.y = 1;
  attr[n].val.clusterDim.z = 1;
  n++;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Launch with thread-block clusters of cluster_x CTAs along x (and programmatic dependent launch if pdl).
template <typename P>
static cudaError_t launch_cluster_x(bool pdl, int cluster_x, cudaStream_t stream, void (*kernel)(P), dim3 grid,
                                    dim3 block, size_t smem, const P &arg) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  attr[n].id = cudaLaunchAttributeClusterDimension;
  attr[n].val.clusterDim.x = (unsigned)cluster_x;
  attr[n].val.clusterDim.y = 1;
  attr[n].val.clusterDim.z = 1;
  n++;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, arg);
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_ex(bool pdl, int cluster_z, cudaStream_t stream, void (*kernel)(KArgs...), dim3 grid,
                             dim3 block, size_t smem, Args... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  if (cluster_z > 1) {  // thread-block clusters along z
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = (unsigned)cluster_z;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

#define LAUNCH_PDL(dev, kernel, grid, block, smem, ...)                                          \
  do {                                                                                           \
    CK(launch_ex((dev)->pdl, 0, (dev)->stream, kernel, dim3(grid), dim3(block), (smem), __VA_ARGS__)); \
    (dev)->launches++;                                                                           \
  } while (0)

// Makes the handle's GPU the current one.
int32_t use(wgpt_device *dev);

// Grows the library-owned workspace (dev->scratch) to at least this many bytes; not while a pass list is being recorded.
int32_t scratch_reserve(wgpt_device *dev, size_t bytes);

// Calls that synchronise the stream (or free memory a recording may name) are not valid while a pass list is
// being recorded: a synchronise on a capturing stream would invalidate the capture.
#define NOT_RECORDING(dev, what)                                                                       \
  REQUIRE(!(dev)->capturing, WGPT_ERR_STATE, "%s is not valid between wgpt_graph_begin and wgpt_graph_end", what)
