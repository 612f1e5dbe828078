// Host-side helpers shared by the library's translation units: CUDA error
// checks, per-device facts, launch profiling and stream-ordered scratch.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <stdexcept>
#include <string>
#include <vector>

namespace mlxvs_b200 {

inline void check_cuda(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw std::runtime_error(std::string("[mlxvs_b200] CUDA error: ") + cudaGetErrorString(e) +
                             " (" + what + ")");
  }
}
#define CK(x) check_cuda((x), #x)

inline void require(bool ok, const std::string& msg) {
  if (!ok) throw std::invalid_argument(msg);
}

struct DeviceInfo {
  int sms = 0;
  int max_smem = 0;
  uint32_t* err = nullptr;  // error word of the kernels' bounded waits
  size_t total_mem = 0;     // device memory in bytes
};

inline DeviceInfo& device_info() {
  static std::mutex mu;
  static DeviceInfo infos[64];
  static bool ready[64] = {};
  int dev = 0;
  CK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64)
    throw std::runtime_error("[mlxvs_b200] device ordinal " + std::to_string(dev) +
                             " is beyond the 64 devices this library tracks");
  std::lock_guard<std::mutex> guard(mu);
  DeviceInfo& info = infos[dev];
  if (!ready[dev]) {
    int major = 0, minor = 0;
    CK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    CK(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev));
    if (major != 10 || minor != 0)
      throw std::runtime_error("[mlxvs_b200] needs an sm_100 GPU (B200); device " +
                               std::to_string(dev) + " is sm_" + std::to_string(major) +
                               std::to_string(minor));
    CK(cudaDeviceGetAttribute(&info.sms, cudaDevAttrMultiProcessorCount, dev));
    CK(cudaDeviceGetAttribute(&info.max_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
    {
      size_t free_b = 0;
      CK(cudaMemGetInfo(&free_b, &info.total_mem));
    }
    CK(cudaMalloc(&info.err, 16));
    CK(cudaMemset(info.err, 0, 16));
    // keep freed scratch in this process's pool between calls
    cudaMemPool_t pool;
    CK(cudaDeviceGetDefaultMemPool(&pool, dev));
    uint64_t keep = UINT64_MAX;
    CK(cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep));
    ready[dev] = true;
  }
  return info;
}

// ------------------------------------------------------------- profiling
// When enabled, every launch of the library's kernels is bracketed by CUDA
// events recorded on the launching stream; profile_read sums their device
// times per kernel name.  Off by default (benchmarks turn it on).
struct ProfRecord {
  const char* name;
  cudaEvent_t start, stop;
  double issued;  // tensor-core operations the launch issued (0: none)
};
inline std::mutex prof_mu;
inline bool prof_on = false;
inline std::vector<ProfRecord> prof_records;

struct ProfScope {
  const char* name;
  cudaStream_t s;
  cudaEvent_t start = nullptr, stop = nullptr;
  double issued = 0.0;
  ProfScope(const char* n, cudaStream_t st) : name(n), s(st) {
    bool on;
    {
      std::lock_guard<std::mutex> g(prof_mu);
      on = prof_on;
    }
    if (!on) return;
    CK(cudaEventCreate(&start));
    CK(cudaEventCreate(&stop));
    CK(cudaEventRecord(start, s));
  }
  ~ProfScope() {
    if (!start) return;
    cudaEventRecord(stop, s);
    std::lock_guard<std::mutex> g(prof_mu);
    prof_records.push_back({name, start, stop, issued});
  }
};

// Scratch buffers of one call, returned to the pool in stream order.
struct Scratch {
  cudaStream_t s;
  std::vector<void*> ptrs;
  explicit Scratch(cudaStream_t st) : s(st) {}
  template <class T>
  T* alloc(size_t count) {
    void* p = nullptr;
    CK(cudaMallocAsync(&p, std::max<size_t>(count * sizeof(T), 256), s));
    ptrs.push_back(p);
    return static_cast<T*>(p);
  }
  ~Scratch() {
    for (void* p : ptrs) cudaFreeAsync(p, s);
  }
};

// Bounded waits inside the kernels give up after this long (no legitimate
// wait comes near it: stages turn over in microseconds).
constexpr uint64_t WAIT_LIMIT_NS = 2000000000ull;

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link
// against libcuda).
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  if (!fn) throw std::runtime_error("[mlxvs_b200] cuTensorMapEncodeTiled is unavailable");
  return fn;
}

}  // namespace mlxvs_b200
