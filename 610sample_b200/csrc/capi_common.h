// What the files of the C ABI share: per-thread error text and launch count, the device's status word (attn_capi.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_b200.h"

namespace attn {
namespace capi {

// stores the message of an error and returns its code
int fail(int code, const char* fmt, ...);
// binds the current device's context to this thread; its status word
int begin(unsigned int** status);
// the end of an entry point that has launched `launches` kernels
int done(cudaError_t e, const char* what, const char* why, int launches);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace capi
}  // namespace attn
