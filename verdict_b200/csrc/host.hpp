// Host-side helpers shared by the library's translation units: errors that
// cross the C ABI as codes, CUDA call checks and the driver's tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <exception>
#include <mutex>
#include <string>

#include "vdexec.h"

namespace vd {

struct VdError {
  int code;
  std::string msg;
};

[[noreturn]] inline void fail(int code, const std::string& msg) { throw VdError{code, msg}; }

inline void cuda_check(cudaError_t e, const char* what) {
  if (e != cudaSuccess) fail(VD_ECUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

inline void put_err(char* err, size_t errlen, const std::string& msg) {
  if (!err || errlen == 0) return;
  const size_t n = std::min(errlen - 1, msg.size());
  std::memcpy(err, msg.data(), n);
  err[n] = '\0';
}

// Runs the body of a C entry point that has no handle; nothing thrown leaves it.
template <class F>
int guarded_call(char* err, size_t errlen, F&& body) noexcept {
  try {
    body();
    return VD_OK;
  } catch (const VdError& e) {
    put_err(err, errlen, e.msg);
    return e.code;
  } catch (const std::exception& e) {
    put_err(err, errlen, e.what());
    return VD_EINVAL;
  } catch (...) {
    put_err(err, errlen, "unknown error");
    return VD_EINVAL;
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  if (!fn) fail(VD_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  return fn;
}

}  // namespace vd
