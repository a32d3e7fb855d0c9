// mev_internal.h -- what the translation units of libmev.so share beside the C ABI.
#ifndef MEV_INTERNAL_H_
#define MEV_INTERNAL_H_

#include <hip/hip_runtime.h>

#include "mev.h"

// Keeps the text of a failed HIP call for mev_last_hip_error (thread-local).
__attribute__((visibility("hidden"))) void mev_note_hip_error(const char* file, int line,
                                                             const char* call, hipError_t e);

#define MEV_HIP(call)                                     \
  do {                                                    \
    hipError_t _e = (call);                               \
    if (_e != hipSuccess) {                               \
      mev_note_hip_error(__FILE__, __LINE__, #call, _e);  \
      return MEV_EHIP;                                    \
    }                                                     \
  } while (0)

#endif  // MEV_INTERNAL_H_
