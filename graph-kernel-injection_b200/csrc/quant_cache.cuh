// Device view of an 8-bit ring cache (format in quant_cache.cu) and what the shared-prefix
// entry points need of it.
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

// One attend call.  The result goes to o (16 bits, LSE 0 for an empty sequence) or, where o32 is
// given, unrounded to o32 with LSE -inf for an empty sequence.
struct QAttend {
  const void* q;
  const void *k, *v, *scales;
  const int64_t* lengths;
  void* o;
  float *o32, *lse;
  int64_t B, H, kv_heads, d;
  int dtype, fmt;
  double scale;
  int64_t sink, window;
  cudaStream_t stream;
};
int qcache_attend_check(const QAttend& a);   // an SBFA_ERR_* code; launches nothing
int qcache_attend_launch(const QAttend& a);  // after the check

}  // namespace sbfa
