// ssm_host.hpp — host helpers of the selective state space block's entry
// points.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "dwconv1d_host.hpp"
#include "pathtile_hip.h"

namespace pt {

inline bool ssm_aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline long long ssm_ceil(long long n, long long q) { return (n + q - 1) / q; }
inline size_t ssm_round(size_t n) { return (n + 63) / 64 * 64; }

// Launches `blocks` workgroups: a grid's lanes count up to 2^32 - 1.
inline int ssm_launch(const void* fn, long long blocks, int threads, void* stream, void** args) {
  if (blocks == 0) return PT_OK;
  if (blocks < 0 || blocks * threads >= (1LL << 32)) return PT_ERR_SHAPE;
  return launch(fn, (uint32_t)blocks, (uint32_t)threads, 0, stream, args);
}

}  // namespace pt
