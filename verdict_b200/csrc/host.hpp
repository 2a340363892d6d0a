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

// cuTensorMapEncodeTiled, which wants a context current on the calling thread:
// where no runtime call has made one so yet, that of the thread's device.
struct EncodeTiled {
  EncodeTiledFn fn = nullptr;
  template <class... A>
  CUresult operator()(const A&... a) const {
    CUresult r = fn(a...);
    if (r == CUDA_ERROR_INVALID_CONTEXT) {
      int dev = 0;
      cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
      cuda_check(cudaSetDevice(dev), "cudaSetDevice");
      r = fn(a...);
    }
    return r;
  }
};

inline EncodeTiled encode_fn() {
  static EncodeTiled encode;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      encode.fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  if (!encode.fn) fail(VD_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  return encode;
}

}  // namespace vd
