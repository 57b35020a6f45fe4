// Host helpers shared by the library's C entry points.
#pragma once

#include <stdint.h>

namespace piper {

// Records the text piper_last_error() returns on this thread; returns `status`.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Compute units and XCCs of the current device (looked up once per device).
int device_topology(int* cus, int* xccs);

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

}  // namespace piper
