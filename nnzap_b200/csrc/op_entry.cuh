// What the C entry points of the operators on device pointers share.
#pragma once
#include <cuda_runtime.h>

#include <string>

#include "../../include/nnz_b200.h"

namespace nnz {

void set_last_error(const std::string& msg);      // engine.cu
// The current device's error word and its number of SMs (engine.cu).
int op_device(int** err, int* num_sms);

// No C++ exception crosses the C ABI: building the message can throw.
inline int refuse(int code, const char* what) noexcept {
  try {
    set_last_error(what);
  } catch (...) {
  }
  return code;
}

inline int cuda_rc(cudaError_t e, const char* who) noexcept {
  if (e == cudaSuccess) return NNZ_OK;
  try {
    set_last_error(std::string(who) + ": " + cudaGetErrorString(e));
  } catch (...) {
  }
  return NNZ_ECUDA;
}

}  // namespace nnz
