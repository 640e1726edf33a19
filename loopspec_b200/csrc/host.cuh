// Host-side pieces shared by the library's translation units: the exception
// that carries an LS_E* code to the C entry points, the check macros, the
// kernel launch wrapper and the handle-less error text.
#pragma once

#include <cuda_runtime.h>

#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/loopspec_engine.h"

namespace ls {

struct EngineError : std::runtime_error {
  int code;
  EngineError(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

#define CK(x)                                                                            \
  do {                                                                                   \
    cudaError_t e_ = (x);                                                                \
    if (e_ != cudaSuccess)                                                               \
      throw ::ls::EngineError(LS_ECUDA, std::string(#x) + ": " + cudaGetErrorString(e_));      \
  } while (0)

#define REQUIRE(cond, code, msg)                  \
  do {                                                \
    if (!(cond)) throw ::ls::EngineError((code), (msg));    \
  } while (0)

// Records the text of a failed call that has no engine handle (read with
// ls_last_error(NULL), per thread) and returns its LS_E* code.
int fail_global(const std::exception& ex);

// Launch with optional programmatic-dependent-launch attribute.
template <typename... KArgs, typename... Args>
void launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl,
            Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl ? attr : nullptr;
  cfg.numAttrs = pdl ? 1 : 0;
  CK(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

}  // namespace ls
