// Library-wide entry points: version, thread-local error string, device checks.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace fdk {

static thread_local char g_last_error[512] = "no error";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FDK_ERR_LAUNCH, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return FDK_OK;
}

// Per-device attributes, cached; host threads may race on the first query (each writes the same
// values, the count before the major that marks the slot filled).
static std::atomic<int> g_sm_major[64];
static std::atomic<int> g_sm_count[64];

static int query(int dev) {
  if (dev < 0 || dev >= 64) return FDK_ERR_DEVICE;
  if (g_sm_major[dev].load(std::memory_order_acquire) == 0) {
    int major = 0, count = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      return FDK_ERR_DEVICE;
    }
    g_sm_count[dev].store(count, std::memory_order_relaxed);
    g_sm_major[dev].store(major, std::memory_order_release);
  }
  return FDK_OK;
}

// (kernel, device) pairs whose dynamic shared-memory limit has been raised; guarded by a mutex so
// concurrent first calls from several host threads each see the attribute set before launching.
static std::mutex g_attr_mu;
static const void* g_attr_func[256];
static int g_attr_dev[256];
static int g_attr_n = 0;

int ensure_smem_attr(const void* func, int bytes, const char* what) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return set_error(FDK_ERR_DEVICE, "%s: no current device", what);
  }
  std::lock_guard<std::mutex> lock(g_attr_mu);
  for (int i = 0; i < g_attr_n; ++i)
    if (g_attr_func[i] == func && g_attr_dev[i] == dev) return FDK_OK;
  const cudaError_t e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(FDK_ERR_LAUNCH, "%s: cannot set %d bytes of shared memory: %s", what, bytes, cudaGetErrorString(e));
  }
  if (g_attr_n < 256) {
    g_attr_func[g_attr_n] = func;
    g_attr_dev[g_attr_n] = dev;
    ++g_attr_n;
  }
  return FDK_OK;
}

int check_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return set_error(FDK_ERR_DEVICE, "no CUDA device available");
  }
  if (query(dev) != FDK_OK) return set_error(FDK_ERR_DEVICE, "cannot query CUDA device %d", dev);
  const int major = g_sm_major[dev].load(std::memory_order_acquire);
  if (major != 10)
    return set_error(FDK_ERR_DEVICE, "device %d is sm_%d0; this library is built for sm_100a only", dev, major);
  return FDK_OK;
}

int sm_count() {
  int dev = 0;
  cudaGetDevice(&dev);
  if (query(dev) != FDK_OK) return 148;
  return g_sm_count[dev].load(std::memory_order_relaxed);
}

}  // namespace fdk

extern "C" const char* fdk_version(void) { return "fastdecisions-b200 0.1.0 sm_100a"; }

extern "C" const char* fdk_get_last_error_string(void) { return fdk::g_last_error; }

namespace fdk {

// One 64-bit slot as an argument of type T.
template <typename T>
static T slot_as(const char* args, size_t i) {
  int64_t raw;
  memcpy(&raw, args + 8 * i, 8);  // the block has no alignment of its own
  if constexpr (std::is_floating_point_v<T>) {
    double d;
    memcpy(&d, &raw, 8);
    return static_cast<T>(d);
  } else if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(raw));
  } else {
    return static_cast<T>(raw);
  }
}

template <typename... A, size_t... I>
static int invoke(int (*fn)(A...), const char* args, std::index_sequence<I...>) {
  return fn(slot_as<A>(args, I)...);
}

template <typename... A>
static int invoke(int (*fn)(A...), const void* args, int64_t nargs) {
  if (!args || nargs != (int64_t)sizeof...(A))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "invoke: %d arguments expected, %lld given", (int)sizeof...(A),
                     (long long)nargs);
  return invoke(fn, static_cast<const char*>(args), std::index_sequence_for<A...>{});
}

}  // namespace fdk

extern "C" int fdk_invoke(int op, const void* args, int64_t nargs) {
  switch (op) {
    case FDK_OP_PAGED_KV_WRITE: return fdk::invoke(fdk_paged_kv_write, args, nargs);
    case FDK_OP_PAGED_KV_READ: return fdk::invoke(fdk_paged_kv_read, args, nargs);
    case FDK_OP_PAGED_GQA_FWD: return fdk::invoke(fdk_paged_gqa_fwd, args, nargs);
    case FDK_OP_RECURRENT_GATED_DELTA_RULE_FWD: return fdk::invoke(fdk_recurrent_gated_delta_rule_fwd, args, nargs);
    case FDK_OP_PACKED_CONV_STATE: return fdk::invoke(fdk_packed_conv_state, args, nargs);
    default: return fdk::set_error(FDK_ERR_INVALID_ARGUMENT, "invoke: unknown entry point %d", op);
  }
}
