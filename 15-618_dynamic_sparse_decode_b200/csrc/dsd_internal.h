// dsd_internal.h -- error plumbing shared by the C ABI's translation units.
#pragma once

#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <new>
#include <stdexcept>
#include <string>

#include "dsd_b200.h"

namespace dsd_internal {

inline thread_local std::string g_last_error;

// NVTX range over a host-side phase (entry points, and each stage of the step
// while it is launched or captured), the counterpart of the reference's
// ScopedStageTimer stages in a profiler timeline.  Header-only NVTX: without
// an attached tool each push/pop is a no-op call.
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

struct DsdError {
  int code;
  std::string msg;
};

[[noreturn]] inline void Fail(int code, const std::string& msg) { throw DsdError{code, msg}; }

inline void Check(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    Fail(DSD_ECUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
}

template <typename F>
int Guard(F&& f) {
  try {
    f();
    return DSD_OK;
  } catch (const DsdError& e) {
    g_last_error = e.msg;
    return e.code;
  } catch (const std::bad_alloc&) {
    g_last_error = "host allocation failed";
    return DSD_ENOMEM;
  } catch (const std::exception& e) {
    g_last_error = e.what();
    return DSD_EINVAL;
  } catch (...) {
    g_last_error = "unknown error";
    return DSD_EINVAL;
  }
}

// Makes `device` current for the call and restores the caller's device on
// every exit path (including a failure thrown by Fail/Check).
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int device) {
    Check(cudaGetDevice(&prev), "cudaGetDevice");
    if (prev != device) Check(cudaSetDevice(device), "cudaSetDevice");
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

}  // namespace dsd_internal
