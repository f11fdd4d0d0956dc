// 8-bit StreamingLLM ring cache: write (quantise), attend, read back.
//
// Format.  One sequence b and key/value head h own R = sink + window rows of
// DP codes (DP = head_dim rounded up to 64, 128 or 256; the columns behind
// head_dim hold 0) for K and for V, and one pair of scale bytes (K, V) per
// row.  Row r < sink holds position r, position p >= sink lives in row
// sink + (p - sink) % window.  A row x is stored as codes c and byte e + 127,
//   e = least integer with max|x| <= top * 2^e  (top = 448 e4m3, 127 int8),
//   c = x * 2^-e rounded to the code type, ties to even,
// so the scaling itself is exact, every code carries one rounding, and c * 2^e
// is exact in fp32.  e >= -126; an all-zero row has e = 0.  A row with a NaN
// or an infinity is stored as byte 255 with zero codes and reads as NaN.  A
// code may round a value next to the 16-bit type's largest up past it: what
// is read, and an attention's result, saturates there instead of overflowing.
//
// Every sequence has its own length L on the device, so a batch may be ragged
// and a captured step advances when it is replayed.  The visible rows of the
// query at position L - 1 are always rows [0, min(L, R)): before the ring is
// full they are the positions in order, afterwards all of them are in the
// window or sinks, and attention does not depend on the order of its keys.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>

#include "quant_cache.cuh"
#include "tc_prims.cuh"

namespace sbfa {
namespace {

namespace cg = cooperative_groups;
using tc::ex2;
using tc::smem_u32;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kFull = 0xffffffffu;
constexpr uint32_t kBadRow = 255;   // scale byte of a row with a NaN or an infinity
constexpr uint32_t kZeroByte = 127;   // of a row of zeros (and of others with e = 0)

// ---------------------------------------------------------------------------
// codes and scales
// ---------------------------------------------------------------------------

// Scale byte of a row whose largest magnitude has the fp32 bits `amax`.
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return kBadRow;
  if (amax == 0) return kZeroByte;
  // amax = f * 2^E, f in [1, 2); top = 1.75 * 2^8 or 1.984375 * 2^6
  constexpr int kTopExp = FMT == SBFA_Q_E4M3 ? 8 : 6;
  constexpr uint32_t kTopMant = FMT == SBFA_Q_E4M3 ? 0x600000u : 0x7e0000u;
  const int e = (int)(amax >> 23) - kTopExp + ((amax & 0x7fffffu) > kTopMant ? 1 : 0);
  return (uint32_t)max(e, 1);   // biased; subnormal amax gives e <= 1 as well
}
// 2^(byte - 127); NaN for a bad row.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == kBadRow ? 0x7fc00000u : byte << 23);
}
// 2^(127 - byte), the factor a row is multiplied by before rounding
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}

// Four values (already scaled) to four codes.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (FMT == SBFA_Q_E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  } else {
    // |x| <= 127 by the choice of the scale
    const uint32_t x = (uint32_t)__float2int_rn(a) & 0xffu, y = (uint32_t)__float2int_rn(b) & 0xffu;
    const uint32_t z = (uint32_t)__float2int_rn(c) & 0xffu, w = (uint32_t)__float2int_rn(d) & 0xffu;
    return x | (y << 8) | (z << 16) | (w << 24);
  }
}
// The bits of four codes that are all zero where the codes are: e4m3 has a negative zero.
template <int FMT>
__device__ __forceinline__ constexpr uint32_t code_mask() {
  return FMT == SBFA_Q_E4M3 ? 0x7f7f7f7fu : 0xffffffffu;
}
// Codes 0, 1 (lo) and 2, 3 (hi) of a word as half pairs (exact).
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == SBFA_Q_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // code + 128 in the low byte of a half with exponent 2^10 is 1024 + 128
    // + code exactly; one subtraction leaves the code
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&ha);
    hi = *reinterpret_cast<uint32_t*>(&hb);
  }
}

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}

// x limited to T's finite range (NaN stays)
template <typename T>
__device__ __forceinline__ float saturated(float x) {
  constexpr float top = std::is_same<T, __half>::value ? 65504.f : 3.38953138925153547590e38f;
  return fabsf(x) > top ? copysignf(top, x) : x;
}

// two values rounded to T within its finite range (NaN stays)
template <typename T> __device__ __forceinline__ uint32_t pack2_sat(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2_sat<__half>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2_sat<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A group of 8 lanes (16 at 256 columns) takes one (head, token): pieces of 16 bytes of K and
// of V, the row maxima in packed 16-bit integers (the magnitudes of both 16-bit types are
// ordered like their bits) with one shuffle chain for both, 8 code bytes back per piece. Bound
// by HBM (4 D bytes in, 2 D + 2 out per head and token): 16 x 8 x 2048 rows of 128 take 45 us
// with 16 lanes a row and fp32 maxima, 38.5 us so (and with fewer instructions).  A CTA covers
// 2^hs heads x kRows / 2^hs tokens at a time (tokens adjacent, so that their scale pairs share
// sectors; several heads only where a call has few tokens) and walks the tokens that survive
// the call: positions that a later token of it overwrites are never visited.  The last CTA of a
// sequence moves its length on (a ticket per sequence, left at zero), which saves a second
// launch in every decode step.
constexpr int kAppThreads = 256;
constexpr int kAppCtas = 6;     // resident per SM
constexpr int kAppRounds = 2;   // of them, with at least two passes each
constexpr int app_lanes(int dp) { return dp == 256 ? 16 : 8; }

// fp32 bits of the magnitude whose 16 bits are `h`
template <typename T> __device__ __forceinline__ uint32_t magnitude_bits(uint32_t h);
template <> __device__ __forceinline__ uint32_t magnitude_bits<__nv_bfloat16>(uint32_t h) {
  return h << 16;
}
template <> __device__ __forceinline__ uint32_t magnitude_bits<__half>(uint32_t h) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

template <typename T, int FMT, int DP>
__global__ void __launch_bounds__(kAppThreads, kAppCtas)
    qcache_append_kernel(QCache c, int64_t* __restrict__ lengths, int32_t* __restrict__ tickets,
                         const T* __restrict__ kn, const T* __restrict__ vn, Strides3 sk,
                         Strides3 sv, const int64_t* __restrict__ counts, int n_new,
                         int head_blocks, int hs) {
  constexpr int G = app_lanes(DP);
  constexpr int VPL = DP / (8 * G);                          // pieces of a row per lane
  constexpr int kRows = kAppThreads / G;
  const int b = blockIdx.y;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G;
  const int tp = kRows >> hs;                                // tokens a CTA covers at a time
  const int head = ((int)blockIdx.x % head_blocks << hs) + slot / tp;
  const int chunk = (int)blockIdx.x / head_blocks, chunks = (int)gridDim.x / head_blocks;
  const int64_t len = max(lengths[b], (int64_t)0);
  const int cnt = counts ? (int)min(max(counts[b], (int64_t)0), (int64_t)n_new) : n_new;
  const int sink = (int)c.sink, window = (int)c.window;
  // survivors: tokens [0, n_sink) into rows len + t, tokens [t_win, cnt) into the window
  const int n_sink = (int)max((int64_t)0, min((int64_t)cnt, c.sink - len));
  const int t_win = max(n_sink, cnt - window);
  const int items = n_sink + cnt - t_win;
  const int slot0 = cnt > t_win ? (int)((len + t_win - c.sink) % c.window) : 0;
  const bool real = head < (int)c.heads;
  const T* ks = kn + b * sk.b + head * sk.h + lane * 8;
  const T* vs = vn + b * sv.b + head * sv.h + lane * 8;
  const int64_t row0 = ((int64_t)b * c.heads + head) * c.rows;
  for (int j0 = chunk * tp; j0 < items; j0 += chunks * tp) {
    const int j = j0 + slot % tp;
    uint4 x[2][VPL];
    int row = -1;
#pragma unroll
    for (int i = 0; i < VPL; ++i) x[0][i] = x[1][i] = make_uint4(0, 0, 0, 0);
    if (j < items && real) {
      const int k = j - n_sink;
      const int t = k < 0 ? j : t_win + k;
      const int w = slot0 + k;                               // < 2 * window
      row = k < 0 ? (int)len + j : sink + (w >= window ? w - window : w);
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if ((lane + i * G) * 8 < c.d) {
          x[0][i] = __ldcs(reinterpret_cast<const uint4*>(ks + t * sk.n + i * G * 8));
          x[1][i] = __ldcs(reinterpret_cast<const uint4*>(vs + t * sv.n + i * G * 8));
        }
    }
    uint32_t m[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const uint4 w = x[p][i];
        m[p] = __vmaxu2(m[p], __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu),
                                       __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
      }
    // both rows' maxima in one word: K's in the low half, V's in the high one
    uint32_t both = __vmaxu2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
    for (int s = G / 2; s > 0; s >>= 1)
      both = __vmaxu2(both, __shfl_xor_sync(kFull, both, s, G));
    uint32_t bytes = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint32_t e = scale_byte<FMT>(magnitude_bits<T>(p == 0 ? both & 0xffffu : both >> 16));
      bytes |= e << (8 * p);
      const bool bad = e == kBadRow;
      const float inv = bad ? 0.f : scale_inverse(e);
      const float2 inv2 = make_float2(inv, inv);
      uint8_t* dst = (p == 0 ? c.k : c.v) + (row0 + row) * DP + lane * 8;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const uint4 w = x[p][i];
        const float2 f0 = __fmul2_rn(unpack2<T>(w.x), inv2), f1 = __fmul2_rn(unpack2<T>(w.y), inv2);
        const float2 f2 = __fmul2_rn(unpack2<T>(w.z), inv2), f3 = __fmul2_rn(unpack2<T>(w.w), inv2);
        const uint32_t lo = encode4<FMT>(f0.x, f0.y, f1.x, f1.y);
        const uint32_t hi = encode4<FMT>(f2.x, f2.y, f3.x, f3.y);
        if (row >= 0)
          *reinterpret_cast<uint2*>(dst + i * G * 8) =
              bad ? make_uint2(0, 0) : make_uint2(lo, hi);
      }
    }
    if (row >= 0 && lane == 0) c.scales[row0 + row] = (uint16_t)bytes;
  }
  // every CTA of this sequence has read its length before the last one writes it
  __syncthreads();
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) {
      lengths[b] = len + cnt;
    } else {
      __threadfence();
      if (atomicAdd(&tickets[b], 1) == (int)gridDim.x - 1) {
        tickets[b] = 0;
        lengths[b] = len + cnt;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
// Out row i of a sequence is its i-th kept position in order (sinks, then the window from its
// oldest), rows behind the last one are zero with position -1. A group of DP / 8 lanes per row,
// CTAs walk the rows of one head; bound by HBM (2 D + 2 bytes in, 4 D out per kept row and
// head).  64 x 8 x 2052 rows of 128 took 175, 144, 138, 131 us with 1, 2, 4, 8 rounds of
// resident CTAs (many short ones keep loads and stores of different CTAs apart), and take 128.5
// us since the conversion saturates by itself.
constexpr int kReadThreads = 256;
constexpr int kReadUnroll = 4;
constexpr int kReadRounds = 8;   // of resident CTAs

template <typename T, int FMT>
__device__ __forceinline__ uint4 values8(uint2 codes, float scale) {
  uint32_t h[4];
  decode4<FMT>(codes.x, h[0], h[1]);
  decode4<FMT>(codes.y, h[2], h[3]);
  uint32_t r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __fmul2_rn(__half22float2(*reinterpret_cast<__half2*>(&h[j])),
                                make_float2(scale, scale));
    r[j] = pack2_sat<T>(f.x, f.y);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T, int FMT, int G>
__global__ void __launch_bounds__(kReadThreads)
    qcache_read_kernel(QCache c, const int64_t* __restrict__ lengths, T* __restrict__ ko,
                       T* __restrict__ vo, int64_t* __restrict__ positions, int head_blocks,
                       int hs) {
  constexpr int DP = G * 8;
  constexpr int kRows = kReadThreads / G;
  const int b = blockIdx.y;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G;
  const int tp = kRows >> hs;
  const int head = ((int)blockIdx.x % head_blocks << hs) + slot / tp;
  const int chunk = (int)blockIdx.x / head_blocks, chunks = (int)gridDim.x / head_blocks;
  if (head >= (int)c.heads) return;
  const int64_t len = max(lengths[b], (int64_t)0);
  const int rows = (int)c.rows, sink = (int)c.sink, window = (int)c.window;
  const int kept = (int)min(len, c.rows);
  // behind the sinks, out row i is position shift + i; the oldest of them is in slot0
  const int64_t shift = len <= c.rows ? 0 : len - c.rows;
  const int slot0 = window > 0 ? (int)(shift % c.window) : 0;
  const int64_t row0 = ((int64_t)b * c.heads + head) * c.rows;
  const bool on = lane * 8 < c.d;
  for (int i0 = chunk * tp * kReadUnroll + slot % tp; i0 < rows; i0 += chunks * tp * kReadUnroll) {
    uint2 xk[kReadUnroll], xv[kReadUnroll];
    uint32_t sc[kReadUnroll];
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
      const int i = i0 + u * tp;
      xk[u] = xv[u] = make_uint2(0, 0);
      sc[u] = 0x7f7f;
      if (i < kept) {
        const int w = slot0 + i - sink;                      // < 2 * window
        const int64_t src = row0 + (i < sink ? i : sink + (w >= window ? w - window : w));
        xk[u] = __ldcs(reinterpret_cast<const uint2*>(c.k + src * DP) + lane);
        xv[u] = __ldcs(reinterpret_cast<const uint2*>(c.v + src * DP) + lane);
        sc[u] = c.scales[src];
      }
    }
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
      const int i = i0 + u * tp;
      if (i < rows) {
        if (lane == 0 && head == 0)
          positions[b * c.rows + i] = i >= kept ? -1 : i < sink ? i : shift + i;
        if (on) {
          const int64_t dst = (row0 + i) * c.d + lane * 8;
          __stcs(reinterpret_cast<uint4*>(ko + dst),
                 values8<T, FMT>(xk[u], scale_value(sc[u] & 255u)));
          __stcs(reinterpret_cast<uint4*>(vo + dst),
                 values8<T, FMT>(xv[u], scale_value(sc[u] >> 8)));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// attend (one query position per sequence)
// ---------------------------------------------------------------------------
// O = softmax(scale q K^T) V over rows [0, min(L, R)).  Per key/value head the
// rows are read once for 8 * NQ query heads of its group.  Bound by HBM: 2 D + 2
// bytes per row against 8 * NQ * 4 D operations.
//
// Both products put the cache on the M side of mma.m16n8k16 (fp16 in, fp32 out)
// and the query heads on the N side, which lets every lane load its operands
// straight from global memory in 16-byte pieces, without shared memory:
//   S^T = K Q^T: lane (g, c) = (lane / 4, lane % 4) holds bytes [16 c, 16 c + 16) of
//     each 64-byte piece of rows g and g + 8; the order of the summed d does not
//     matter as long as Q's fragment uses the same one;
//   O^T = V^T P^T: lane (g, c) holds its DP / 8 bytes of rows 2c, 2c + 1, 2c + 8 and
//     2c + 9; byte permutes pair two keys of one d, and the m16 tiles number the d's
//     so that a lane's own columns are its rows g and g + 8.
// P^T comes out of the score fragment with movmatrix.  Codes become fp16 exactly.
//
// Scales: a key's 2^ek multiplies its score in fp32.  A value row's 2^ev is folded
// into the exponent of its weight: P' = 2^(x + ev - M), M a running reference kLift below the largest
// x + ev so far, so P' is at most 2^(kLift + kSlack), just below fp16's largest: a weight times
// scale keeps fp16's 11 bits down to 2^-25 of the largest one and is off by up to 2^-36 of it below.
// The row sum l = sum 2^(x - m) has its own per-lane reference m (both in fp32); the result is
// acc / l * 2^(M - m).  A row of zeros, which has a scale all the same, does not enter M.  Q is
// scaled by a power of two into fp16's range, which is exact for fp16 inputs and for bf16 down to
// 2^-31 of the row's largest element (8 significant bits above fp16's step of 2^-24; smaller
// elements lose their last ones).
//
// Two ways to spread the units (sequence, key/value head, group of queries) over the GPU:
//  - few units: a cluster of NS CTAs shares one, its warps take every (4 NS)-th step of KS
//    rows, warps merge through shared memory and CTAs through distributed shared
//    memory: one launch, no workspace;
//  - many: as many CTAs as fit on the SMs each take an equal run of the steps of all units in order
//    (FLAT), whatever the lengths.  The lengths are only known here, so every CTA sums them
//    up.  A warp fetches its first step of the next unit before the merge of this one, so that
//    loads stay in flight across units.  A unit that crosses from one CTA to the next leaves
//    partial rows that qcache_join_kernel merges, in order.
constexpr int kAttWarps = 4;
constexpr float kSlack = 4.f;   // how far scores may pass a reference before it moves
constexpr float kLift = 11.f;   // 2^(kLift + kSlack) * 448 * rows fits fp32, 2^(kLift + kSlack) fp16

// Resident CTAs per SM that the registers are limited for.  At two sets of query columns steps
// of 32 rows on two CTAs beat steps of 16 on three (64 x 8 heads of 12 queries x 2052 rows: 72
// against 84 us).
constexpr int att_ctas(int dp, int nq) { return dp == 256 || nq == 2 ? 2 : 3; }

template <int DP, int NQ>
struct AttCfg {
  static constexpr int kTiles = DP == 256 ? 1 : 2;   // 16-row tiles per step
  static constexpr int kRowsQ = 8 * NQ;
  static constexpr int kCtas = att_ctas(DP, NQ);
  // per warp: O [8 NQ][DP + 4]; M, m, l [8 NQ]; the CTA's M, m, l
  static constexpr int kPitch = DP + 4;
  static constexpr size_t kBytes =
      ((size_t)kAttWarps * kRowsQ * (kPitch + 3) + 3 * kRowsQ) * sizeof(float);
};

__device__ __forceinline__ uint4 ldg16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ldg8(const uint8_t* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
               : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ldg2(const uint16_t* p) {
  uint16_t r;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// One row's four columns from `parts` partial results: stat(0 | 1 | 2, w) gives M, m, l of part
// w, vec(w) its columns.  Maxima ignore NaN, which comes through the sums.
template <typename S, typename V>
__device__ __forceinline__ void att_join(int parts, S&& stat, V&& vec, float& Mx, float& mx,
                                         float& L, float4& a) {
  Mx = mx = -INFINITY;
  for (int w = 0; w < parts; ++w) {
    Mx = fmaxf(Mx, stat(0, w));
    mx = fmaxf(mx, stat(1, w));
  }
  const float rM = Mx == -INFINITY ? 0.f : Mx, rm = mx == -INFINITY ? 0.f : mx;
  L = 0.f;
  a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < parts; ++w) {
    L += stat(2, w) * ex2(stat(1, w) - rm);
    const float f = ex2(stat(0, w) - rM);
    const float4 p = vec(w);
    a.x += p.x * f;
    a.y += p.y * f;
    a.z += p.z * f;
    a.w += p.w * f;
  }
}

// O (rounded, or fp32 to o32) and LSE of four columns of row `out`; `some`: whether its sequence has
// rows.  Where all their scores are minus infinity L is 0 and the result NaN, with that LSE.
template <typename T>
__device__ __forceinline__ void att_write(T* o, float* o32, float* lse, int64_t out, int d, int col,
                                          bool some, float Mx, float mx, float L, float4 a) {
  const float f = 1.f / L;
  const float back = ex2((Mx == -INFINITY ? 0.f : Mx) - (mx == -INFINITY ? 0.f : mx));
  a.x = some ? a.x * f * back : 0.f;
  a.y = some ? a.y * f * back : 0.f;
  a.z = some ? a.z * f * back : 0.f;
  a.w = some ? a.w * f * back : 0.f;
  if (col < d) {
    if (o32)
      *reinterpret_cast<float4*>(o32 + out * d + col) =
          make_float4(saturated<T>(a.x), saturated<T>(a.y), saturated<T>(a.z), saturated<T>(a.w));
    else
      *reinterpret_cast<uint2*>(o + out * d + col) =
          make_uint2(pack2_sat<T>(a.x, a.y), pack2_sat<T>(a.z, a.w));
  }
  // a partial result marks an empty row by -inf, the public one by 0
  if (col == 0 && lse) lse[out] = some ? (mx + log2f(L)) * kLn2 : (o32 ? -INFINITY : 0.f);
}

// What a CTA of the FLAT form writes for the merge: the unit that its first run ends, if that began
// in an earlier CTA.
struct FlatRecord {
  int64_t unit_start;   // cost of all units before it, -1: nothing to merge
  int64_t total;        // cost of all units
  int64_t row;          // first row of o
  int nq;
};
struct FlatWs {
  FlatRecord* rec;      // [CTAs]
  float* stats;         // [CTAs][2][3][8 NQ] M, m, l
  float* part;          // [CTAs][2][8 NQ][DP]
};
// where the run of CTA i of n begins, in cost from the first unit's start
__device__ __forceinline__ int64_t flat_start(int64_t total, int i, int n) {
  return (int64_t)((uint64_t)total * (uint32_t)i / (uint32_t)n);
}

// A unit costs its steps and about kRunSteps more (its queries, merge and output, and latency
// that one warp step cannot hide): with 2, 4, 8 a ragged batch of 64 x 8 heads of 12 queries
// takes 106, 90, 66 us. Runs are equal in this cost; one that begins in the surplus begins with
// the next unit.
constexpr int kRunSteps = 8;

// A run of steps [s0, s1) of one unit.
struct AttRun {
  int b, hc;            // sequence; (key/value head, group of queries) of it
  int n, steps;         // visible rows and steps of the unit
  int s0, s1;
  int64_t row0;         // first cache row of the unit
};

template <typename T, int FMT, int DP, int NQ, bool FLAT>
__global__ void __launch_bounds__(kAttWarps * 32, (AttCfg<DP, NQ>::kCtas))
    qcache_attend_kernel(const T* __restrict__ q, QCache c, const int64_t* __restrict__ lengths,
                         T* __restrict__ o, float* __restrict__ o32, float* __restrict__ lse,
                         float scale_log2, int group, int chunks, int ns, int batch, bool beside,
                         FlatWs ws) {
  using C = AttCfg<DP, NQ>;
  constexpr int KT = C::kTiles, KS = 16 * KT;
  constexpr int NCH = DP / 64;      // 16-byte pieces of a K row per lane
  constexpr int VW = DP / 32;       // words of a V row per lane
  extern __shared__ __align__(16) float att_smem[];
  tc::griddep_launch();   // what follows (a merge) waits for this kernel's results itself
  // Beside a shared prefix's kernel the last CTA completes after it, and with it this kernel,
  // so that whoever waits for this one has both.  (All CTAs waiting would keep others from
  // starting.)
  auto leave = [&] {
    if (beside && blockIdx.x == gridDim.x - 1) tc::griddep_wait();
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, cc = lane & 3;
  const int hcs = (int)c.heads * chunks;
  auto visible = [&](int b) { return (int)min(max(lengths[b], (int64_t)0), c.rows); };
  // the FLAT form gives an empty sequence a step as well: someone has to write its zeros
  auto steps_of = [&](int n) { return FLAT ? max(1, (n + KS - 1) / KS) : (n + KS - 1) / KS; };
  auto cost_of = [&](int n) { return (int64_t)(steps_of(n) + kRunSteps); };

  // Runs end with the last unit whatever the lengths read later say: a caller's append that races
  // with this call spoils its result, not memory.
  auto last_unit = [&](const AttRun& r) { return r.hc + 1 == hcs && r.b + 1 == batch; };

  AttRun cur;
  int64_t left = 0;       // cost that this CTA takes behind the current unit
  int stride, rank = 0;
  if constexpr (FLAT) {
    __shared__ int64_t scan[kAttWarps];
    __shared__ int first[2];
    // cost of each thread's share of the sequences, and of all before it
    const int per = (batch + kAttWarps * 32 - 1) / (kAttWarps * 32);
    const int b_lo = min((int)threadIdx.x * per, batch), b_hi = min(b_lo + per, batch);
    int64_t mine = 0;
    for (int b = b_lo; b < b_hi; ++b) mine += cost_of(visible(b));
    int64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(kFull, incl, d);
      if (lane >= d) incl += up;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) {
      if (w < warp) incl += scan[w];
      total += scan[w];
    }
    total *= hcs;
    const int64_t begin = flat_start(total, blockIdx.x, gridDim.x);
    const int64_t end = flat_start(total, blockIdx.x + 1, gridDim.x);
    // the sequence in which `begin` falls, and its place there
    __shared__ int64_t inside;
    if (begin >= (incl - mine) * hcs && begin < incl * hcs) {
      int64_t rem = begin - (incl - mine) * hcs;
      int b = b_lo, n = visible(b);
      for (; b + 1 < b_hi && rem >= cost_of(n) * hcs; n = visible(++b)) rem -= cost_of(n) * hcs;
      first[0] = b;
      first[1] = n;
      inside = rem;
    }
    if (threadIdx.x == 0) ws.rec[blockIdx.x].unit_start = -1;
    if (begin == end) {                            // a few short units, more CTAs
      leave();
      return;
    }
    __syncthreads();
    cur.b = first[0];
    cur.n = first[1];
    cur.steps = steps_of(cur.n);
    const int64_t cost = cost_of(cur.n);
    cur.hc = (int)min(inside / cost, (int64_t)hcs - 1);
    const int64_t at = inside - cur.hc * cost;     // place of `begin` in its unit
    cur.s0 = (int)min(at, (int64_t)cur.steps);
    cur.s1 = (int)min((int64_t)cur.steps, at + (end - begin));
    left = max((int64_t)0, end - begin - (cost - at));
    const int64_t unit_start = begin - at;
    if (cur.s0 >= cur.s1) {                        // nothing of that unit: begin with the next
      if (left == 0 || last_unit(cur)) {
        leave();
        return;
      }
      if (++cur.hc == hcs) {
        cur.hc = 0;
        cur.n = visible(++cur.b);
        cur.steps = steps_of(cur.n);
      }
      cur.s0 = 0;
      cur.s1 = (int)min((int64_t)cur.steps, left);
      left = max((int64_t)0, left - cost_of(cur.n));
    }
    stride = kAttWarps;
    if (threadIdx.x == 0 && cur.s0 > 0 && cur.s1 == cur.steps) {
      FlatRecord r;
      r.unit_start = unit_start;
      r.total = total;
      r.row = ((int64_t)cur.b * c.heads + cur.hc / chunks) * group + cur.hc % chunks * C::kRowsQ;
      r.nq = min(C::kRowsQ, group - cur.hc % chunks * C::kRowsQ);
      ws.rec[blockIdx.x] = r;
    }
  } else {
    rank = blockIdx.x % ns;
    const int unit = blockIdx.x / ns;
    cur.b = unit / hcs;
    cur.hc = unit % hcs;
    cur.n = visible(cur.b);
    cur.steps = steps_of(cur.n);
    cur.s0 = rank * kAttWarps;
    cur.s1 = cur.steps;
    stride = ns * kAttWarps;
  }

  uint4 kr[KT][2][NCH];
  uint32_t vr[KT][4][VW];
  uint32_t sc[KT][2], sc_next[KT][2];
  // Rows of step s of a run.  A full step's addresses are one base and constants; in a unit's last
  // step rows behind the last visible one read that one again.
  auto load_k = [&](const AttRun& r, int s) {
    const uint8_t* kb = c.k + r.row0 * DP + cc * 16;
    const uint16_t* sb = c.scales + r.row0;
    if ((s + 1) * KS <= r.n) {
      const int64_t row = s * KS + g;
      kb += row * DP;
      sb += row;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int j = 0; j < NCH; ++j) kr[t][i][j] = ldg16(kb + (t * 16 + i * 8) * DP + j * 64);
          sc_next[t][i] = ldg2(sb + t * 16 + i * 8);
        }
    } else {
      const int last = max(r.n - 1, 0);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t row = min(s * KS + t * 16 + i * 8 + g, last);
#pragma unroll
          for (int j = 0; j < NCH; ++j) kr[t][i][j] = ldg16(kb + row * DP + j * 64);
          sc_next[t][i] = ldg2(sb + row);
        }
    }
  };
  auto load_vrow = [&](uint32_t (&w)[VW], const uint8_t* p) {
    if constexpr (DP == 64) {
      const uint2 x = ldg8(p);
      w[0] = x.x;
      w[1] = x.y;
    } else {
#pragma unroll
      for (int j = 0; j < VW / 4; ++j) {
        const uint4 x = ldg16(p + j * 128);
        w[4 * j] = x.x;
        w[4 * j + 1] = x.y;
        w[4 * j + 2] = x.z;
        w[4 * j + 3] = x.w;
      }
    }
  };
  auto load_v = [&](const AttRun& r, int s) {
    const uint8_t* vb = c.v + r.row0 * DP + g * (DP == 64 ? 8 : 16);
    if ((s + 1) * KS <= r.n) {
      vb += (int64_t)(s * KS + 2 * cc) * DP;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          load_vrow(vr[t][i], vb + (t * 16 + (i >> 1) * 8 + (i & 1)) * DP);
    } else {
      const int last = max(r.n - 1, 0);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = s * KS + t * 16 + (i >> 1) * 8 + 2 * cc + (i & 1);
          load_vrow(vr[t][i], vb + (int64_t)min(row, last) * DP);
        }
    }
  };

  auto first_row = [&](const AttRun& r) {
    return ((int64_t)r.b * c.heads + r.hc / chunks) * c.rows;
  };
  cur.row0 = first_row(cur);
  int s = cur.s0 + warp;
  if (s < cur.s1) {
    load_k(cur, s);
    load_v(cur, s);
  }
  for (;;) {
    // the run behind this one, which starts its unit
    AttRun nxt = cur;
    const bool has_next = FLAT && left > 0 && !last_unit(cur);
    if (has_next) {
      nxt.hc = cur.hc + 1;
      if (nxt.hc == hcs) {
        nxt.hc = 0;
        nxt.b = cur.b + 1;
        nxt.n = visible(nxt.b);
        nxt.steps = steps_of(nxt.n);
      }
      nxt.row0 = first_row(nxt);
      nxt.s0 = 0;
      nxt.s1 = (int)min((int64_t)nxt.steps, left);
      left = max((int64_t)0, left - cost_of(nxt.n));
    }
    const int h0 = cur.hc % chunks * C::kRowsQ;             // first head of the group
    const int nq = min(C::kRowsQ, group - h0);
    const int64_t qrow0 = ((int64_t)cur.b * c.heads + cur.hc / chunks) * group + h0;
    const int n = cur.n;

    // Q fragments, column g of each n-tile, scaled into fp16's range
    uint32_t qf[NQ][DP / 16][2];
    float2 qs[NQ];   // softmax scale (base 2) of the two query columns of this lane
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const int r = t * 8 + g;
      uint32_t raw[NCH][8];
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int hlf = 0; hlf < 2; ++hlf) {
          const int col = j * 64 + cc * 16 + hlf * 8;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (r < nq && col < c.d)
            w = __ldg(reinterpret_cast<const uint4*>(q + (qrow0 + r) * c.d + col));
          raw[j][4 * hlf] = w.x;
          raw[j][4 * hlf + 1] = w.y;
          raw[j][4 * hlf + 2] = w.z;
          raw[j][4 * hlf + 3] = w.w;
        }
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = unpack2<T>(raw[j][i]);
          m = max(m, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
        }
      m = max(m, __shfl_xor_sync(kFull, m, 1));
      m = max(m, __shfl_xor_sync(kFull, m, 2));
      // largest element to [2^14, 2^15); fp16 needs none of it (its own range)
      int e = 0;
      if (sizeof(T) == 2 && !std::is_same<T, __half>::value && m != 0 && m < 0x7f800000u)
        e = max(-120, (int)(m >> 23) - 127 - 14);
      const float f_in = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = unpack2<T>(raw[j][i]);
          qf[t][j * 4 + (i >> 1)][i & 1] = tc::pack2<__half>(f.x * f_in, f.y * f_in);
        }
      const float f_out = __uint_as_float((uint32_t)(127 + e) << 23) * scale_log2;
      qs[t] = make_float2(__shfl_sync(kFull, f_out, (2 * cc) * 4),
                          __shfl_sync(kFull, f_out, (2 * cc + 1) * 4));
    }

    float acc[NQ][2 * VW][4];
    float2 M[NQ], m[NQ], l[NQ];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
#pragma unroll
      for (int i = 0; i < 2 * VW; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][i][e] = 0.f;
      M[t] = m[t] = make_float2(-FLT_MAX, -FLT_MAX);   // below every score, and finite
      l[t] = make_float2(0.f, 0.f);
    }

    // whether the loads of this warp's first step in the next run are under way
    const bool into = has_next && warp < nxt.s1;
    bool ahead = false;
    for (; s < cur.s1; s += stride) {
      const bool more = s + stride < cur.s1;
      // S^T, one 16-row tile of keys by 8 query columns each
      float x[NQ][KT][4];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        sc[t][0] = sc_next[t][0];
        sc[t][1] = sc_next[t][1];
#pragma unroll
        for (int u = 0; u < NQ; ++u) x[u][t][0] = x[u][t][1] = x[u][t][2] = x[u][t][3] = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
          const uint32_t w0[4] = {kr[t][0][j].x, kr[t][0][j].y, kr[t][0][j].z, kr[t][0][j].w};
          const uint32_t w1[4] = {kr[t][1][j].x, kr[t][1][j].y, kr[t][1][j].z, kr[t][1][j].w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            decode4<FMT>(w0[w], a0, a2);
            decode4<FMT>(w1[w], a1, a3);
#pragma unroll
            for (int u = 0; u < NQ; ++u)
              mma_f16(x[u][t], a0, a1, a2, a3, qf[u][j * 4 + w][0], qf[u][j * 4 + w][1]);
          }
        }
      }
      if (more) {
        load_k(cur, s + stride);
      } else if (into) {
        load_k(nxt, warp);
      }
      // the scale of the keys' scores and the exponent of their values' (NaN for a bad row)
      float ks[KT][2], ev[KT][2];
      bool maybe_zero = false;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t vbyte = sc[t][i] >> 8;
          ks[t][i] = scale_value(sc[t][i] & 255u);
          ev[t][i] = vbyte == kBadRow ? __uint_as_float(0x7fc00000u) : (float)((int)vbyte - 127);
          maybe_zero |= vbyte == kZeroByte;
        }
      // A value row of zeros shares its byte with rows whose largest value is next to the top code.
      // It adds nothing to O, so its weight must not set the others' reference either: an attention
      // sink of zeros 10 powers of two above values of 2^-10 left none of their bits.  (Where every
      // row has this byte, 64 x 32 heads x 2052 rows take 184 us instead of 176.)
      if (__any_sync(kFull, maybe_zero)) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          uint32_t holds[4];   // lanes that hold a code other than 0 of their row i
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t any = 0;
#pragma unroll
            for (int w = 0; w < VW; ++w) any |= vr[t][i][w];
            holds[i] = __ballot_sync(kFull, (any & code_mask<FMT>()) != 0);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {   // row g + 8 i is row 2 i + g % 2 of the lanes with cc = g / 2
            const uint32_t row = g & 1 ? holds[2 * i + 1] : holds[2 * i];
            if (sc[t][i] >> 8 == kZeroByte && (row & (0x11111111u << (g >> 1))) == 0)
              ev[t][i] = -INFINITY;
          }
        }
      }
      const bool edge = (s + 1) * KS > n;
      // Online softmax; element e of a tile is key g + 8 (e / 2), query 2 cc + e % 2, and the two
      // queries go through packed fp32 pairs.  Both references only move when a score passes what
      // they hold by more than kSlack (rare behind the first steps), which a warp votes on once.
      uint32_t pb[NQ][KT][2];
#pragma unroll
      for (int u = 0; u < NQ; ++u) {
        float2 xs[KT][2], ys[KT][2];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            xs[t][i] = __fmul2_rn(make_float2(x[u][t][2 * i], x[u][t][2 * i + 1]),
                                  __fmul2_rn(qs[u], make_float2(ks[t][i], ks[t][i])));
            ys[t][i] = __fadd2_rn(xs[t][i], make_float2(ev[t][i], ev[t][i]));
          }
        if (edge) {
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (s * KS + t * 16 + i * 8 + g >= n)
                xs[t][i] = ys[t][i] = make_float2(-INFINITY, -INFINITY);
        }
        float2 mx = xs[0][0], my = ys[0][0];
#pragma unroll
        for (int t = 0; t < KT; ++t) {   // maxima ignore NaN
          mx.x = tc::max3f(mx.x, xs[t][0].x, xs[t][1].x);
          mx.y = tc::max3f(mx.y, xs[t][0].y, xs[t][1].y);
          my.x = tc::max3f(my.x, ys[t][0].x, ys[t][1].x);
          my.y = tc::max3f(my.y, ys[t][0].y, ys[t][1].y);
        }
        const bool grow = mx.x > m[u].x + kSlack || mx.y > m[u].y + kSlack ||
                          my.x > M[u].x + (kLift + kSlack) || my.y > M[u].y + (kLift + kSlack);
        if (__any_sync(kFull, grow)) {
          // the row sum's reference is this lane's own
          const float2 mn = make_float2(fmaxf(m[u].x, mx.x), fmaxf(m[u].y, mx.y));
          l[u].x *= ex2(m[u].x - mn.x);
          l[u].y *= ex2(m[u].y - mn.y);
          m[u] = mn;
          // the accumulator's is shared by the warp's keys of a query
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            my.x = fmaxf(my.x, __shfl_xor_sync(kFull, my.x, d));
            my.y = fmaxf(my.y, __shfl_xor_sync(kFull, my.y, d));
          }
          const float2 Mn =
              make_float2(fmaxf(M[u].x, my.x - kLift), fmaxf(M[u].y, my.y - kLift));
          const float2 f = make_float2(ex2(M[u].x - Mn.x), ex2(M[u].y - Mn.y));
          M[u] = Mn;
#pragma unroll
          for (int i = 0; i < 2 * VW; ++i) {
            acc[u][i][0] *= f.x;
            acc[u][i][1] *= f.y;
            acc[u][i][2] *= f.x;
            acc[u][i][3] *= f.y;
          }
        }
        const float2 nm = make_float2(-m[u].x, -m[u].y), nM = make_float2(-M[u].x, -M[u].y);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 a = __fadd2_rn(xs[t][i], nm), b = __fadd2_rn(ys[t][i], nM);
            l[u] = __fadd2_rn(l[u], make_float2(ex2(a.x), ex2(a.y)));
            pb[u][t][i] = movmatrix(tc::pack2<__half>(ex2(b.x), ex2(b.y)));
          }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t a[2][4];   // the word's four columns make two m16 tiles
          decode4<FMT>(__byte_perm(vr[t][0][w], vr[t][1][w], 0x5140), a[0][0], a[0][1]);
          decode4<FMT>(__byte_perm(vr[t][2][w], vr[t][3][w], 0x5140), a[0][2], a[0][3]);
          decode4<FMT>(__byte_perm(vr[t][0][w], vr[t][1][w], 0x7362), a[1][0], a[1][1]);
          decode4<FMT>(__byte_perm(vr[t][2][w], vr[t][3][w], 0x7362), a[1][2], a[1][3]);
#pragma unroll
          for (int u = 0; u < NQ; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              mma_f16(acc[u][2 * w + i], a[i][0], a[i][1], a[i][2], a[i][3], pb[u][t][0],
                      pb[u][t][1]);
        }
      if (more) {
        load_v(cur, s + stride);
      } else if (into) {
        load_v(nxt, warp);
        ahead = true;
      }
    }
    if (into && !ahead) {   // a warp without a step in this run
      load_k(nxt, warp);
      load_v(nxt, warp);
    }

    // ---- merge: lanes, then warps, then the CTAs of the cluster
    float* so = att_smem;                                         // [warp][row][kPitch]
    float* sM = so + kAttWarps * C::kRowsQ * C::kPitch;           // [warp][row] M, m, l
    float* sm = sM + kAttWarps * C::kRowsQ;
    float* sl = sm + kAttWarps * C::kRowsQ;
#pragma unroll
    for (int u = 0; u < NQ; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mi = i == 0 ? m[u].x : m[u].y, li = i == 0 ? l[u].x : l[u].y;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          const float m2 = __shfl_xor_sync(kFull, mi, d);
          const float l2 = __shfl_xor_sync(kFull, li, d);
          const float mn = fmaxf(mi, m2);
          li = li * ex2(mi - mn) + l2 * ex2(m2 - mn);
          mi = mn;
        }
        const int row = warp * C::kRowsQ + u * 8 + 2 * cc + i;
        if (g == 0) {
          sM[row] = i == 0 ? M[u].x : M[u].y;
          sm[row] = mi;
          sl[row] = li;
        }
        // lane g's columns: word w, bytes 2 t, 2 t + 1 (m16 tile t of the word)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const int col = DP == 64 ? g * 8 + 4 * w : (w >> 2) * 128 + g * 16 + 4 * (w & 3);
          *reinterpret_cast<float4*>(so + row * C::kPitch + col) =
              make_float4(acc[u][2 * w][i], acc[u][2 * w][2 + i], acc[u][2 * w + 1][i],
                          acc[u][2 * w + 1][2 + i]);
        }
      }
    __syncthreads();
    // the CTA's warps into warp 0's place (each thread its own four columns of a row); maxima
    // ignore NaN, which comes through the sums
    float* cM = sl + kAttWarps * C::kRowsQ;   // [row] M, m, l of the CTA
    float* cm = cM + C::kRowsQ;
    float* cl = cm + C::kRowsQ;
    auto write = [&](int row, int col, float Mx, float mx, float L, float4 a) {
      att_write<T>(o, o32, lse, qrow0 + row, c.d, col, n > 0, Mx, mx, L, a);
    };
    for (int idx = threadIdx.x; idx < nq * (DP / 4); idx += kAttWarps * 32) {
      const int row = idx / (DP / 4), col = idx % (DP / 4) * 4;
      float* mine = so + row * C::kPitch + col;
      float Mx, mx, L;
      float4 a;
      att_join(kAttWarps,
               [&](int k, int w) { return sM[(k * kAttWarps + w) * C::kRowsQ + row]; },
               [&](int w) { return *reinterpret_cast<float4*>(mine + w * C::kRowsQ * C::kPitch); },
               Mx, mx, L, a);
      const bool whole = FLAT ? cur.s0 == 0 && cur.s1 == cur.steps : ns == 1;
      if (whole) {
        write(row, col, Mx, mx, L, a);
      } else if constexpr (FLAT) {
        // the end of a unit (slot 0), or its beginning (slot 1)
        const int64_t slot = 2 * (int64_t)blockIdx.x + (cur.s0 > 0 ? 0 : 1);
        *reinterpret_cast<float4*>(ws.part + (slot * C::kRowsQ + row) * DP + col) = a;
        if (col == 0) {
          float* st = ws.stats + slot * 3 * C::kRowsQ + row;
          st[0] = Mx;
          st[C::kRowsQ] = mx;
          st[2 * C::kRowsQ] = L;
        }
      } else {
        *reinterpret_cast<float4*>(mine) = a;
        if (col == 0) {
          cM[row] = Mx;
          cm[row] = mx;
          cl[row] = L;
        }
      }
    }
    if constexpr (!FLAT) {
      if (ns == 1) {
        leave();
        return;
      }
      // the CTAs of the cluster: each takes its share of the rows' columns from all of them
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      for (int idx = rank * (kAttWarps * 32) + threadIdx.x; idx < nq * (DP / 4);
           idx += ns * kAttWarps * 32) {
        const int row = idx / (DP / 4), col = idx % (DP / 4) * 4;
        float Mx, mx, L;
        float4 a;
        att_join(ns,
                 [&](int k, int w) {
                   return *cluster.map_shared_rank(cM + k * C::kRowsQ + row, w);
                 },
                 [&](int w) {
                   return *reinterpret_cast<float4*>(
                       cluster.map_shared_rank(so + row * C::kPitch + col, w));
                 },
                 Mx, mx, L, a);
        write(row, col, Mx, mx, L, a);
      }
      cluster.sync();   // peers may still read this CTA's memory
      leave();
      return;
    }
    if (!has_next) {
      leave();
      return;
    }
    __syncthreads();    // the merge has read what the next run's will overwrite
    cur = nxt;
    s = warp;
  }
}

// Joins the partial rows of the units that cross CTAs of the FLAT form: block i those of the unit
// that ends in CTA i, from the CTA in which it began.  kJoinWarps / rows warps share a row's parts
// (a long sequence among short ones may have hundreds), then the row's first warp joins theirs.
constexpr int kJoinWarps = 16;

template <typename T, int DP, int NQ>
__global__ void __launch_bounds__(kJoinWarps * 32)
    qcache_join_kernel(T* __restrict__ o, float* __restrict__ o32, float* __restrict__ lse, int d,
                       int ctas, FlatWs ws) {
  using C = AttCfg<DP, NQ>;
  constexpr int VEC = DP / 32;   // columns of a lane
  __shared__ float so[kJoinWarps][DP];
  __shared__ float st[3][kJoinWarps];
  tc::griddep_launch();
  tc::griddep_wait();
  const FlatRecord r = ws.rec[blockIdx.x];
  if (r.unit_start < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int last = blockIdx.x;
  // the last CTA whose run does not begin behind the unit
  int j0 = (int)((uint64_t)r.unit_start * (uint32_t)ctas / (uint64_t)r.total);
  while (j0 + 1 < ctas && flat_start(r.total, j0 + 1, ctas) <= r.unit_start) ++j0;
  while (j0 > 0 && flat_start(r.total, j0, ctas) > r.unit_start) --j0;
  // the CTAs between the two are whole inside the unit; where there are more CTAs than cost,
  // some of them had nothing and left nothing
  const int parts = last - j0 + 1;
  auto slot = [&](int w) { return w == 0 ? 2 * (int64_t)j0 + 1 : 2 * (int64_t)(j0 + w); };
  int share = kJoinWarps;        // warps of a row
  while (share * r.nq > kJoinWarps) share >>= 1;
  const int row = warp / share, part0 = warp % share;
  float Mx = -INFINITY, mx = -INFINITY, L = 0.f;
  float a[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) a[i] = 0.f;
  // (M, m, l, columns) of another part joined to (Mx, mx, L, a)
  auto add = [&](float M2, float m2, float l2, const float* v) {
    const float Mn = fmaxf(Mx, M2), mn = fmaxf(mx, m2);
    const float rM = Mn == -INFINITY ? 0.f : Mn, rm = mn == -INFINITY ? 0.f : mn;
    L = L * ex2(mx - rm) + l2 * ex2(m2 - rm);
    const float f1 = ex2(Mx - rM), f2 = ex2(M2 - rM);
#pragma unroll
    for (int i = 0; i < VEC; ++i) a[i] = a[i] * f1 + v[i] * f2;
    Mx = Mn;
    mx = mn;
  };
  if (row < r.nq) {
#pragma unroll 4
    for (int w = part0; w < parts; w += share) {
      if (r.total < ctas &&
          flat_start(r.total, j0 + w, ctas) == flat_start(r.total, j0 + w + 1, ctas))
        continue;
      const float* p = ws.stats + slot(w) * 3 * C::kRowsQ + row;
      const float* src = ws.part + (slot(w) * C::kRowsQ + row) * DP + lane * VEC;
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i += 2)
        *reinterpret_cast<float2*>(v + i) = *reinterpret_cast<const float2*>(src + i);
      add(p[0], p[C::kRowsQ], p[2 * C::kRowsQ], v);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) so[warp][lane * VEC + i] = a[i];
    if (lane == 0) {
      st[0][warp] = Mx;
      st[1][warp] = mx;
      st[2][warp] = L;
    }
  }
  __syncthreads();
  if (row >= r.nq || part0 != 0) return;
  for (int w = warp + 1; w < warp + min(share, parts); ++w)
    add(st[0][w], st[1][w], st[2][w], &so[w][lane * VEC]);
#pragma unroll
  for (int i = 0; i < VEC; i += 4) {
    const int col = lane * VEC + i;
    if constexpr (VEC >= 4) {
      att_write<T>(o, o32, lse, r.row + row, d, col, true, Mx, mx, L,
                   make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]));
    } else {   // two columns a lane: even lanes write their neighbour's as well
      const float2 up = make_float2(__shfl_down_sync(kFull, a[0], 1),
                                    __shfl_down_sync(kFull, a[1], 1));
      if (lane % 2 == 0)
        att_write<T>(o, o32, lse, r.row + row, d, col, true, Mx, mx, L,
                     make_float4(a[0], a[1], up.x, up.y));
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int padded_dim(int64_t d) {
  if (d <= 0 || d > 256 || d % 8 != 0) return 0;
  return d <= 64 ? 64 : d <= 128 ? 128 : 256;
}

// Geometry of a cache (no pointers).
int check_geometry(const sbfa_qcache* c) {
  if (c == nullptr) return fail(SBFA_ERR_INVALID, "8-bit cache: NULL cache");
  if (c->dtype != SBFA_F16 && c->dtype != SBFA_BF16)
    return fail(SBFA_ERR_UNSUPPORTED, "8-bit cache: dtype must be float16 or bfloat16");
  if (c->fmt != SBFA_Q_E4M3 && c->fmt != SBFA_Q_INT8)
    return fail(SBFA_ERR_INVALID, "8-bit cache: unknown format code");
  if (c->batch <= 0 || c->kv_heads <= 0)
    return fail(SBFA_ERR_INVALID, "batch and kv_heads must be positive");
  if (c->batch > 65535 || c->kv_heads >= (1 << 24))
    return fail(SBFA_ERR_UNSUPPORTED, "8-bit cache: at most 65535 sequences and 2^24 heads");
  if (padded_dim(c->head_dim) == 0)
    return fail(SBFA_ERR_UNSUPPORTED,
                "8-bit cache: head_dim must be a multiple of 8 and at most 256");
  if (c->sink < 0 || c->window < 0)
    return fail(SBFA_ERR_INVALID, "sink_size and window_size must be non-negative");
  if (c->sink >= (1ll << 30) || c->window >= (1ll << 30) || c->sink + c->window <= 0 ||
      c->sink + c->window >= (1ll << 30))
    return fail(SBFA_ERR_INVALID, "sink_size + window_size must be in [1, 2^30)");
  return SBFA_OK;
}

int check_qcache(const sbfa_qcache* c) {
  if (int rc = check_geometry(c)) return rc;
  if (!c->k_codes || !c->v_codes || !c->scales || !c->lengths)
    return fail(SBFA_ERR_INVALID, "8-bit cache: NULL cache tensor");
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15u)
    return fail(SBFA_ERR_INVALID, "8-bit cache: tensors must be 16-byte aligned");
  return SBFA_OK;
}

QCache device_view(const sbfa_qcache* c) {
  return QCache{(uint8_t*)c->k_codes, (uint8_t*)c->v_codes, (uint16_t*)c->scales, c->kv_heads,
                c->sink + c->window, c->sink, c->window, (int)c->head_dim};
}

template <typename F>
int by_format(int dtype, int fmt, int64_t D, F&& f) {
  // f(type tag, format, padded dim) with the last two as integral constants
  auto dims = [&](auto t, auto m) {
    switch (padded_dim(D)) {
      case 64: return f(t, m, std::integral_constant<int, 64>{});
      case 128: return f(t, m, std::integral_constant<int, 128>{});
      default: return f(t, m, std::integral_constant<int, 256>{});
    }
  };
  auto fmts = [&](auto t) {
    return fmt == SBFA_Q_E4M3 ? dims(t, std::integral_constant<int, SBFA_Q_E4M3>{})
                              : dims(t, std::integral_constant<int, SBFA_Q_INT8>{});
  };
  return dtype == SBFA_BF16 ? fmts(__nv_bfloat16{}) : fmts(__half{});
}

// Grid of the append and read kernels for `rows` rows of each head: 2^hs heads per CTA
// where a head has fewer rows than a CTA takes at a time, else as many CTAs along a head as
// make `ctas` per SM in all, each with at least `passes` passes.  (One token of 8 sequences with
// 8 heads: 2.8 us with the heads in one CTA, 3.5 with a CTA each.)
struct RowGrid {
  dim3 grid;
  int head_blocks, hs;
};
int row_grid(int64_t B, int64_t H, int64_t rows, int per_cta, int unroll, int passes, int ctas,
             RowGrid* g) {
  int hs = 0;
  while ((1 << (hs + 1)) <= per_cta && (1 << hs) < H && (per_cta >> (hs + 1)) >= rows) ++hs;
  const int64_t blocks = (H + (1ll << hs) - 1) >> hs;
  const int64_t step = (int64_t)(per_cta >> hs) * unroll * passes;
  const int64_t want = (int64_t)device_sm_count() * ctas;
  const int64_t chunks = std::max<int64_t>(
      1, std::min((rows + step - 1) / step, (want + B * blocks - 1) / (B * blocks)));
  if (blocks * chunks >= (1ll << 31))
    return fail(SBFA_ERR_UNSUPPORTED, "8-bit cache: too many heads");
  g->grid = dim3((unsigned)(blocks * chunks), (unsigned)B);
  g->head_blocks = (int)blocks;
  g->hs = hs;
  return SBFA_OK;
}

// How a call's units are spread over the GPU.
struct AttPlan {
  int nq;               // groups of 8 query heads per CTA
  int chunks;           // groups of 8 nq heads in a key/value head's group
  bool flat;
  int grid, ns;         // CTAs; CTAs of a cluster
  int64_t ws_bytes;
};
int attend_plan(int64_t B, int64_t kv_heads, int64_t group, int64_t d, int64_t rows, int busy_sms,
                AttPlan* p) {
  const int dp = padded_dim(d);
  // 16 query columns halve the passes over a group of more than 8; at 256 columns per row
  // the second set of accumulators would not fit the registers
  p->nq = dp <= 128 && group > 8 ? 2 : 1;
  const int rows_q = 8 * p->nq;
  p->chunks = (int)((group + rows_q - 1) / rows_q);
  const int64_t units = B * kv_heads * p->chunks;
  if (units >= (1ll << 27) || kv_heads * p->chunks >= (1ll << 27))
    return fail(SBFA_ERR_UNSUPPORTED, "8-bit cache: too many (sequence, head) units");
  const int64_t slots = (int64_t)(device_sm_count() - busy_sms) * att_ctas(dp, p->nq);
  // A cluster shortens a unit while there are SMs to fill (8 heads x 1028 rows: 12.4, 9.7, 7.6,
  // 6.9 us on 1, 2, 4, 8 CTAs a unit), with some steps for each of its warps.
  p->ns = 1;
  while (p->ns < 8 && units * p->ns * 2 <= slots && rows > (int64_t)p->ns * 128) p->ns *= 2;
  // What its last, partly filled wave costs in rows of a CTA beyond an equal share; the FLAT
  // form's scan and second kernel cost 4 to 5 us, about what 960 rows of 128 bytes take.  64 x 8
  // heads x 2048 rows (two waves) 62 -> 52 us, 8 x 8 x 16384 60 -> 51; 64 x 8 x 256 would go from
  // 12 to 17, 16 x 8 x 2048 from 19 to 22.
  const int64_t waves = (units * p->ns + slots - 1) / slots;
  const int64_t lost = waves * rows / p->ns - units * rows / slots;
  // Beside a prefix's kernel SMs come free meanwhile, so a last wave costs about half of that.
  p->flat = lost * dp > 960 * 128 * (busy_sms > 0 ? 2 : 1);
  p->grid = p->flat ? (int)slots : (int)(units * p->ns);
  if (p->flat) p->ns = 1;
  p->ws_bytes = p->flat ? slots * ((int64_t)sizeof(FlatRecord) +
                                   2 * rows_q * (dp + 3) * (int64_t)sizeof(float))
                        : 0;
  return SBFA_OK;
}

template <typename T, int FMT, int DP, int NQ, bool FLAT>
int launch_attend(const QAttend& a, const QCache& c, const AttPlan& p) {
  using C = AttCfg<DP, NQ>;
  auto kern = qcache_attend_kernel<T, FMT, DP, NQ, FLAT>;
  static_assert(C::kBytes <= 48 * 1024, "more shared memory than a launch gets unasked");
  FlatWs ws = {};
  ws.rec = (FlatRecord*)a.ws;
  ws.stats = (float*)(ws.rec + p.grid);
  ws.part = ws.stats + (int64_t)p.grid * 2 * 3 * C::kRowsQ;
  const int group = (int)(a.H / c.heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.grid);
  cfg.blockDim = dim3(kAttWarps * 32);
  cfg.dynamicSmemBytes = C::kBytes;
  cfg.stream = a.stream;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (p.ns > 1) {
    cudaLaunchAttribute& x = at[cfg.numAttrs++];
    x.id = cudaLaunchAttributeClusterDimension;
    x.val.clusterDim.x = (unsigned)p.ns;
    x.val.clusterDim.y = x.val.clusterDim.z = 1;
  }
  if (a.beside) {
    cudaLaunchAttribute& x = at[cfg.numAttrs++];
    x.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    x.val.programmaticStreamSerializationAllowed = 1;
  }
  {
    LaunchScope ls("qcache_attend_kernel", a.stream);
    if (int rc = check_cuda(
            cudaLaunchKernelEx(&cfg, kern, (const T*)a.q, c, (const int64_t*)a.cache->lengths,
                               (T*)a.o, a.o32, a.lse, (float)a.scale * kLog2e, group, p.chunks, p.ns,
                               (int)a.cache->batch, a.beside, ws),
            "qcache_attend_kernel"))
      return rc;
  }
  if constexpr (FLAT) {
    LaunchScope ls("qcache_join_kernel", a.stream);
    return check_cuda(launch_early(qcache_join_kernel<T, DP, NQ>, (unsigned)p.grid,
                                   kJoinWarps * 32, 0, a.stream, true, (T*)a.o, a.o32, a.lse,
                                   c.d, p.grid, ws),
                      "qcache_join_kernel");
  }
  return SBFA_OK;
}

}  // namespace
}  // namespace sbfa

using namespace sbfa;

extern "C" int64_t sbfa_qcache_row_bytes(int64_t head_dim) { return padded_dim(head_dim); }

extern "C" int sbfa_qcache_append(const sbfa_qcache* cache, const void* k_new, const void* v_new,
                                  const int64_t* strides, const int64_t* counts, int64_t n_new,
                                  void* stream) {
  if (int rc = check_qcache(cache)) return rc;
  if (n_new < 0 || n_new >= (1ll << 31))
    return fail(SBFA_ERR_INVALID, "sbfa_qcache_append: n_new must be in [0, 2^31)");
  if (n_new == 0) return SBFA_OK;
  if (!k_new || !v_new || !cache->tickets)
    return fail(SBFA_ERR_INVALID, "sbfa_qcache_append: NULL tensor pointer");
  const int64_t H = cache->kv_heads, d = cache->head_dim;
  Strides3 st[2];
  for (int i = 0; i < 2; ++i) {
    st[i] = strides ? Strides3{strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}
                    : Strides3{H * n_new * d, n_new * d, d};
    if (st[i].b < 0 || st[i].h < 0 || st[i].n < 0 || st[i].b % 8 || st[i].h % 8 || st[i].n % 8)
      return fail(SBFA_ERR_INVALID, "sbfa_qcache_append: strides must be non-negative multiples "
                                    "of 8 elements");
  }
  if (((uintptr_t)k_new | (uintptr_t)v_new) & 15u)
    return fail(SBFA_ERR_INVALID, "sbfa_qcache_append: tensors must be 16-byte aligned");
  const QCache c = device_view(cache);
  cudaStream_t s = (cudaStream_t)stream;
  return by_format(cache->dtype, cache->fmt, d, [&](auto t, auto m, auto dp) {
    using T = decltype(t);
    RowGrid g;
    if (int rc = row_grid(cache->batch, H, std::min(n_new, c.rows),
                          kAppThreads / app_lanes(dp.value), 1, 2, kAppCtas * kAppRounds, &g))
      return rc;
    LaunchScope ls("qcache_append_kernel", s);
    qcache_append_kernel<T, m.value, dp.value><<<g.grid, kAppThreads, 0, s>>>(
        c, cache->lengths, cache->tickets, (const T*)k_new, (const T*)v_new, st[0], st[1], counts,
        (int)n_new, g.head_blocks, g.hs);
    return check_launch("qcache_append_kernel");
  });
}

extern "C" int sbfa_qcache_read(const sbfa_qcache* cache, void* k_out, void* v_out,
                                int64_t* positions, void* stream) {
  if (int rc = check_qcache(cache)) return rc;
  if (!k_out || !v_out || !positions)
    return fail(SBFA_ERR_INVALID, "sbfa_qcache_read: NULL tensor pointer");
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15u)
    return fail(SBFA_ERR_INVALID, "sbfa_qcache_read: tensors must be 16-byte aligned");
  const QCache c = device_view(cache);
  cudaStream_t s = (cudaStream_t)stream;
  return by_format(cache->dtype, cache->fmt, cache->head_dim, [&](auto t, auto m, auto dp) {
    using T = decltype(t);
    constexpr int G = dp.value / 8;
    RowGrid g;
    if (int rc = row_grid(cache->batch, c.heads, c.rows, kReadThreads / G, kReadUnroll, 1,
                          4 * kReadRounds, &g))
      return rc;
    LaunchScope ls("qcache_read_kernel", s);
    qcache_read_kernel<T, m.value, G><<<g.grid, kReadThreads, 0, s>>>(
        c, cache->lengths, (T*)k_out, (T*)v_out, positions, g.head_blocks, g.hs);
    return check_launch("qcache_read_kernel");
  });
}

namespace sbfa {
// The plan of a call over H query heads.
static int plan_for(const sbfa_qcache* c, int64_t H, int busy_sms, AttPlan* p) {
  if (H <= 0 || H % c->kv_heads != 0)
    return fail(SBFA_ERR_INVALID, "the query head count must be a multiple of kv_heads");
  if (H / c->kv_heads >= (1 << 20)) return fail(SBFA_ERR_UNSUPPORTED, "too many query heads");
  return attend_plan(c->batch, c->kv_heads, H / c->kv_heads, c->head_dim, c->sink + c->window,
                     busy_sms, p);
}

int64_t qcache_attend_ws_bytes(const sbfa_qcache* cache, int64_t H, int busy_sms) {
  AttPlan p;
  if (check_geometry(cache) != SBFA_OK || plan_for(cache, H, busy_sms, &p) != SBFA_OK) return -1;
  return p.ws_bytes;
}

int qcache_attend_check(const QAttend& a) {
  if (int rc = check_qcache(a.cache)) return rc;
  if (!(a.scale > 0) || a.scale > 1e30)
    return fail(SBFA_ERR_INVALID, "softmax_scale must be positive and finite");
  if (!a.q || (!a.o && !a.o32))
    return fail(SBFA_ERR_INVALID, "8-bit cache: NULL query or output pointer");
  if (((uintptr_t)a.q | (uintptr_t)a.o | (uintptr_t)a.o32 | (uintptr_t)a.ws) & 15u)
    return fail(SBFA_ERR_INVALID, "8-bit cache: tensors must be 16-byte aligned");
  AttPlan p;
  if (int rc = plan_for(a.cache, a.H, a.busy_sms, &p)) return rc;
  if (p.ws_bytes > 0 && (a.ws == nullptr || a.ws_bytes < p.ws_bytes))
    return fail(SBFA_ERR_INVALID, "8-bit cache: workspace too small (need " +
                                      std::to_string(p.ws_bytes) + " bytes)");
  return SBFA_OK;
}

int qcache_attend_launch(const QAttend& a) {
  const QCache c = device_view(a.cache);
  AttPlan p;
  if (int rc = plan_for(a.cache, a.H, a.busy_sms, &p)) return rc;
  return by_format(a.cache->dtype, a.cache->fmt, a.cache->head_dim, [&](auto t, auto m, auto dp) {
    using T = decltype(t);
    constexpr int DP = dp.value;
    if constexpr (DP <= 128) {
      if (p.nq == 2)
        return p.flat ? launch_attend<T, m.value, DP, 2, true>(a, c, p)
                      : launch_attend<T, m.value, DP, 2, false>(a, c, p);
    }
    return p.flat ? launch_attend<T, m.value, DP, 1, true>(a, c, p)
                  : launch_attend<T, m.value, DP, 1, false>(a, c, p);
  });
}
}  // namespace sbfa

extern "C" int64_t sbfa_qcache_attend_workspace_bytes(const sbfa_qcache* cache, int64_t H) {
  return qcache_attend_ws_bytes(cache, H, 0);
}

extern "C" int sbfa_qcache_attend(const sbfa_qcache* cache, const void* q, void* o, float* lse,
                                  int64_t H, double softmax_scale, void* ws, int64_t ws_bytes,
                                  void* stream) {
  const QAttend a{cache, q, o, nullptr, lse, H, softmax_scale, ws, ws_bytes,
                  false, 0, (cudaStream_t)stream};
  if (int rc = qcache_attend_check(a)) return rc;
  return qcache_attend_launch(a);
}
