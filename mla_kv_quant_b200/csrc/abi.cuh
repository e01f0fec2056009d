// Argument checks and error messages shared by the C entry points (abi.cu, int4_abi.cu).
#pragma once

#include <cstdint>

namespace rolaq {

// Records the message that rolaq_last_error() returns on this host thread; returns `code`.
int fail(int code, const char* fmt, ...);

// A launcher's status: ROLAQ_ECUDA gets the runtime's message.
int cuda_rc(int rc, const char* what);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace rolaq
