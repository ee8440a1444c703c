// Host helpers of the training operators' launchers: pieces of a workspace, and early returns.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "../../include/mamba3_b200.h"

namespace m3b {

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Takes 256-byte aligned pieces in order; of a null base it only counts the bytes.
struct Carve {
  uint8_t* base;
  size_t at = 0;
  explicit Carve(void* p) : base(static_cast<uint8_t*>(p)) {}
  void* take(size_t bytes) {
    void* r = base ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return r;
  }
};

}  // namespace m3b

// Return the status of a call that failed.
#define M3B_TRY(x)                     \
  do {                                 \
    const int rc_ = (x);               \
    if (rc_ != M3B_OK) return rc_;     \
  } while (0)
