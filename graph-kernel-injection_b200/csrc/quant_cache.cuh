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
  const sbfa_qcache* cache;
  const void* q;
  void* o;
  float *o32, *lse;
  int64_t H;
  double scale;
  void* ws;
  int64_t ws_bytes;
  // Whether the kernel ahead in the stream is a shared prefix's, beside which this call may run: it
  // starts early, and does not complete before that one has.
  bool beside;
  int busy_sms;   // that the prefix's kernel takes meanwhile
  cudaStream_t stream;
};
// Scratch of a call, -1 for a bad shape.
int64_t qcache_attend_ws_bytes(const sbfa_qcache* cache, int64_t H, int busy_sms);
int qcache_attend_check(const QAttend& a);   // an SBFA_ERR_* code; launches nothing
int qcache_attend_launch(const QAttend& a);  // after the check

// A launch whose kernel may start before the kernel ahead of it in the stream has ended (and
// waits for it itself).
template <typename... P, typename... A>
cudaError_t launch_early(void (*kern)(P...), unsigned grid, unsigned block, size_t smem,
                         cudaStream_t s, bool early, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace sbfa
