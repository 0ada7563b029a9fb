// tm_internal.h -- helpers shared by the library's translation units (not part of the ABI).
#ifndef TM_INTERNAL_H
#define TM_INTERNAL_H

#include <stdint.h>

// Records a formatted message for tm_last_error() (thread-local) and returns `code`.
__attribute__((visibility("hidden"))) int tm_internal_fail(int code, const char* fmt, ...);

// TM_OK, or TM_EINVAL with a message where a call's tensor and chunk tables or the chunk size cannot be.
__attribute__((visibility("hidden"))) int tm_internal_check_table(const void* d_tensors, int64_t n_tensors,
                                                                  const void* d_chunks, int64_t n_chunks,
                                                                  int64_t chunk_elems, const char* who);

#endif
