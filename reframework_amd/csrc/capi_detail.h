// What the extern "C" entry points of capi.hip and capi_mx.hip share: the calling
// thread's error message and the checks of arguments.
#pragma once

#include "common.h"

namespace moe355 {

// Keeps the message for moe355_last_error and returns code.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int check_hip(hipError_t e, const char* what);

inline size_t align256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

inline bool valid_dtype(int d) { return d == MOE355_F32 || d == MOE355_BF16 || d == MOE355_F16; }

inline int elem_size(int d) { return d == MOE355_F32 ? 4 : 2; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

template <typename T>
T* at(void* ws, size_t off) {
  return reinterpret_cast<T*>(static_cast<char*>(ws) + off);
}

}  // namespace moe355
