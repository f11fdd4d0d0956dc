// Device view of an 8-bit ring cache (format in quant_cache.cu).
#pragma once

#include <type_traits>

#include "sbfa_common.cuh"

namespace sbfa {

int device_sm_count();

struct QCache {
  uint8_t* k;         // [B][heads][rows][DP] codes
  uint8_t* v;
  uint16_t* scales;   // [B][heads][rows], K's byte low, V's high
  int64_t heads, rows, sink, window;
  int d;              // head_dim <= DP
};

}  // namespace sbfa
