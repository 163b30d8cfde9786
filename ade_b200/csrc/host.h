// What the translation units of the library share on the host side; nothing here is exported.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ade_host __attribute__((visibility("hidden"))) {

bool cuda_ok(cudaError_t e);            // false and remembered for ade_b200_last_cuda_error if e is an error
int sm_count(int* sms);                 // ADE_OK and the current device's SM count, or why the kernels cannot run on it
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace ade_host
