// Host side of the 8-bit products, shared by the dense and the expert entry
// points.
#pragma once

#include <atomic>
#include <utility>

#include "mtc_internal.h"

namespace mtc {
namespace fp8 {

// One product over token tiles ("slots", mtc_fp8.cuh): a dense matrix, or the
// matrices of several experts.  The tokens are either codes with scales
// (xq), or activations that the kernel quantizes itself (X, 16 rows per slot
// at most).  A gate / up pair leaves act(gate) * up as codes and scales.
struct Product {
  const mtc_fp8_matrix* w[2] = {nullptr, nullptr};  // w[1]: the up matrix of a gate / up pair
  const int32_t* slots = nullptr;                   // device slot list, or null for a dense product
  int experts = 0;                                  // > 0: slots are the expert ids of one token's rows
  int slot_bound = 0;                               // slots of the launch at most
  int rows = 0;                                     // rows of the token operand
  int tile = 128;                                   // rows per slot
  bool many = false;                                // 128 tokens x 256 features per tile
  const uint8_t* xq = nullptr;
  long long ldq = 0;
  const float* sx = nullptr;
  long long lds = 0;
  const void* X = nullptr;
  int xdt = 0;
  long long ldx = 0;
  const int32_t* order = nullptr;
  int kdiv = 1;
  int gate_act = 0;
  void* Y = nullptr;
  int ydt = 0;
  long long ldy = 0;
  const float* bias = nullptr;
  int act = 0;
  uint8_t* hq = nullptr;                            // with w[1]: quantized act(gate) * up
  long long ldh = 0;
  float* hs = nullptr;
  long long hs_ld = 0;
  bool early = false;                               // the weights (and slots) may be read before the predecessor ends
  uint32_t* status = nullptr;
};

// Rows of an operand, and tiles of a product, at most: indexes of rows, of
// tiles and of the blocks behind the last one stay below 2^31.
constexpr long long kMaxRows = 0x7fff0000ll;

int check_matrix(const mtc_fp8_matrix* w, const char* who);

inline bool type_ok(int dt) { return dt == MTC_F32 || dt == MTC_BF16 || dt == MTC_F16; }
// Whether p is aligned to elements of that type (fp32, or 4-byte words).
inline bool aligned(const void* p, int dt = MTC_F32) {
  return (reinterpret_cast<uintptr_t>(p) & (dt == MTC_F32 ? 3 : 1)) == 0;
}
int sm_count();

// Launch with programmatic stream serialization: the kernel may start while
// its predecessor in the stream still runs.  Every kernel launched like this
// calls griddep_wait() before its first access to global memory that the
// predecessor may have written or still reads, and
// griddep_launch_dependents() only after that: so whatever was enqueued
// before the predecessor has completed when a kernel starts, and may be read
// before its griddep_wait().
template <typename... Params, typename... Args>
cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// The dynamic shared-memory limit of a kernel, raised once per device.
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// How many clusters of `cluster` CTAs the device holds at once, one CTA per
// SM: fewer than its SMs allow by number (15 of 8, 33 of 4 on 148 SMs), since
// a cluster stays inside one GPC.  Asked once per device; 0 if unknown.
constexpr int kMaxCluster = 8;
typedef std::atomic<int> ClusterCounts[64][kMaxCluster + 1];
template <typename Kernel>
int resident_clusters(Kernel kernel, int threads, size_t smem, int cluster, ClusterCounts& known) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 0;
  if ((n = known[dev][cluster].load(std::memory_order_relaxed)) > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  known[dev][cluster].store(n, std::memory_order_relaxed);
  return n;
}
int launch_product(const Product& a, cudaStream_t st, const char* who);

// Rows of activations to codes and scales; with `pos` row m goes to the rows
// pos[m * copies ..] that are not negative.
struct QuantRows {
  const void* X = nullptr;
  int dt = 0, M = 0, K = 0;
  long long ldx = 0;
  const int32_t* pos = nullptr;
  int copies = 1;
  uint8_t* q = nullptr;
  long long ldq = 0;
  float* s = nullptr;
  long long lds = 0;
};
int launch_quantize(const QuantRows& a, cudaStream_t st, const char* who);

}  // namespace fp8
}  // namespace mtc
