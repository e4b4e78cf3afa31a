// checks.h -- a failed call's status and message, for the C entry points.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/senmoe.h"
#include "kernels.h"

namespace senmoe {

inline int reject(int status, const char* fmt, ...) {
  char buf[384];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_failure(status, buf);
}

inline int cuda_status(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return SENMOE_OK;
  return reject(e == cudaErrorNotSupported ? SENMOE_ERR_UNSUPPORTED : SENMOE_ERR_CUDA, "%s: %s", what,
                cudaGetErrorString(e));
}

}  // namespace senmoe
