// Error boundary and buffer checks shared by the C entry points.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <exception>
#include <new>
#include <string>

#include "layout.h"

namespace t0b {

inline void Message(char* error, size_t size, const char* text) {
  if (error != nullptr && size != 0) std::snprintf(error, size, "tensor0-b200: %s", text);
}

// Run `body`, mapping invalid arguments to 1 and everything else to 2.
template <typename Body>
int Guard(char* error, size_t size, Body&& body) {
  try {
    body();
    return 0;
  } catch (const InvalidArgument& e) {
    Message(error, size, e.what());
    return 1;
  } catch (const std::bad_alloc&) {
    Message(error, size, "out of host memory");
    return 2;
  } catch (const std::exception& e) {
    Message(error, size, e.what());
    return 2;
  } catch (...) {
    Message(error, size, "unknown exception");
    return 2;
  }
}

inline uint64_t Bytes(uint64_t elements, uint64_t item) {
  uint64_t out = 0;
  if (!CheckedMul(elements, item, &out) || out > static_cast<uint64_t>(PTRDIFF_MAX)) {
    throw InvalidArgument("buffer size exceeds addressable storage");
  }
  return out;
}

// The reference's overlap rule (ffi/buffers.h:43-52).
inline void Disjoint(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  if (a_bytes == 0 || b_bytes == 0) return;
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const bool overlap = x <= y ? y - x < a_bytes : x - y < b_bytes;
  if (overlap) throw InvalidArgument("input and output buffers overlap");
}

}  // namespace t0b
