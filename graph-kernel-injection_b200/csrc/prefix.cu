// Attention of a batch to a prefix that all its sequences share.
//
// Every query sees every prefix token, so the n_q query rows of all B sequences and
// of the G query heads of a key/value head form one matrix of R = B G n_q rows per
// key/value head: O_p = softmax(scale Q K^T) V with K, V read once for the batch
// instead of once per sequence.  Row r is (sequence, head of the group, query) =
// (r / (G n_q), r / n_q % G, r % n_q).
//
// prefix_tc_kernel: one CTA per (256 rows, key/value head, slice of the keys), the
// pipeline of the block-sparse forward without its masks: a TMA warp streams K and V tiles
// of 128 keys through a ring, one warp per 128-row tile issues the MMAs, a warpgroup
// per tile runs the online softmax on TMEM (see attn_tc.cu for the TMEM plan).  Q
// rows come from scattered places, so the softmax threads gather them (a thread per
// row) into the swizzled operand tile.  With 128 rows or fewer in the
// CTA the second tile's warps leave at once.  Few rows against a long prefix are
// bound by HBM (4 D bytes per key) and the key axis is split over the SMs; many rows are
// bound by the tensor cores (4 D operations per row and key).
// Each slice leaves its unnormalised O row in fp32 with (m, l) of its softmax.
//
// prefix_merge_kernel: one warp per query row joins the slices and the row's
// attention over its own tokens (already normalised, with its log-sum-exp).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "tc_attn_common.cuh"

namespace sbfa {

int device_sm_count();

namespace {

using namespace tc;

constexpr int kTM = 128;   // rows per tile (one TMEM lane per row)
constexpr int kPair = 2;   // tiles per CTA
constexpr int kTN = 128;   // keys per K/V tile
constexpr int kHalf = 64;  // keys per half-step (one S slot)
constexpr int kThreads = 384;
constexpr int kRegsCtl = 88;
constexpr int kRegsSoftmax = 208;  // 128*88 + 256*208 == 384*168
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleLog2 = 8.0f;
constexpr uint32_t kTmemCols = 512;

struct PrefixGeom {
  int64_t rows;        // R, rows per key/value head
  int64_t sb, sh, sn;  // q strides (batch, head, query)
  int64_t P;
  int group, n_q, kv_heads, d, splits, n_tiles;
};

template <int D, int STAGES>
struct PrefixLayout {
  static constexpr uint32_t kTile = kTM * D * 2;
  static constexpr uint32_t Q = 0;
  static constexpr uint32_t KV = Q + kPair * kTile;
  static constexpr uint32_t BAR = KV + STAGES * kTile;
  static constexpr int kQFull = 0;
  static constexpr int kKVFull = 1;
  static constexpr int kKVEmpty = 1 + STAGES;
  static constexpr int kSFull = 1 + 2 * STAGES;   // [4], (tile, slot)
  static constexpr int kPFull = 5 + 2 * STAGES;   // [4]
  static constexpr int kPVDone = 9 + 2 * STAGES;  // [2]
  static constexpr int kOFull = 11 + 2 * STAGES;  // [2]
  static constexpr int kDrain = 13 + 2 * STAGES;  // [2]
  static constexpr int kNumBars = 15 + 2 * STAGES;
  static constexpr uint32_t MISC = BAR + kNumBars * 8;
  static constexpr uint32_t kAlloc = MISC + 16 + 1024;
};

template <typename T, int D, int STAGES>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tc_kernel(const T* __restrict__ q, const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, float* __restrict__ part,
                     float2* __restrict__ stats, float scale_log2, PrefixGeom geo, int* status) {
  using L = PrefixLayout<D, STAGES>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescQK = idesc_f16(kBF16, kTM, kHalf, false, false);
  constexpr uint32_t kIdescPV = idesc_f16(kBF16, kTM, D, false, true);
  constexpr int kBoxes = D / 64;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sb = smem_u32(smem);
  auto bar = [&](int i) -> uint32_t { return sb + L::BAR + 8u * (uint32_t)i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y;
  const int64_t row0 = (int64_t)blockIdx.x * kPair * kTM;
  const int nx = row0 + kTM < geo.rows ? 2 : 1;  // tiles with rows in them
  const int split = blockIdx.z;
  // slices of n_tiles / splits tiles, none empty (splits <= n_tiles)
  const int t0 = (int)((int64_t)split * geo.n_tiles / geo.splits);
  const int n = (int)((int64_t)(split + 1) * geo.n_tiles / geo.splits) - t0;

  if (threadIdx.x == 0) {
    mbar_init(bar(L::kQFull), 128 * nx);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar(L::kKVFull + s), 1);
      mbar_init(bar(L::kKVEmpty + s), nx);
    }
    for (int x = 0; x < kPair; ++x) {
      mbar_init(bar(L::kSFull + 2 * x), 1);
      mbar_init(bar(L::kSFull + 2 * x + 1), 1);
      mbar_init(bar(L::kPFull + 2 * x), 128);
      mbar_init(bar(L::kPFull + 2 * x + 1), 128);
      mbar_init(bar(L::kPVDone + x), 1);
      mbar_init(bar(L::kOFull + x), 1);
      mbar_init(bar(L::kDrain + x), 1);
    }
    *abort_flag = 0;
    mbar_init_fence();
    // K_0 and V_0 on their way before the TMEM allocation and the CTA-wide sync
    for (int part_ = 0; part_ < 2; ++part_) {
      mbar_expect_tx(bar(L::kKVFull + part_), L::kTile);
      for (int r = 0; r < kBoxes; ++r)
        tma_load_4d(sb + L::KV + part_ * L::kTile + r * 16384u, part_ == 0 ? &tmk : &tmv,
                    bar(L::kKVFull + part_), 64 * r, t0 * kTN, kvh, 0);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    regs_dec<kRegsCtl>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      int issued = 2;  // entry 2j = K_j, 2j + 1 = V_j
      bool ok = true;
      for (int j = 1; ok && j < n; ++j) {
        for (int part_ = 0; part_ < 2; ++part_) {
          const int e = 2 * j + part_;
          const int s = e % STAGES, f = e / STAGES;
          if (f > 0 &&
              !wait_bar(bar(L::kKVEmpty + s), (uint32_t)((f - 1) & 1), abort_flag, status)) {
            ok = false;
            break;
          }
          mbar_expect_tx(bar(L::kKVFull + s), L::kTile);
          for (int r = 0; r < kBoxes; ++r)
            tma_load_4d(sb + L::KV + s * L::kTile + r * 16384u, part_ == 0 ? &tmk : &tmv,
                        bar(L::kKVFull + s), 64 * r, (t0 + j) * kTN, kvh, 0);
          issued = e + 1;
        }
      }
      for (int s = 0; s < STAGES; ++s) {  // our own copies still in flight
        const int fills = issued > s ? (issued - 1 - s) / STAGES + 1 : 0;
        if (fills) wait_bar_drain(bar(L::kKVFull + s), (uint32_t)((fills - 1) & 1), status);
      }
    } else if ((warp == 1 || warp == 2) && warp <= nx) {
      // ---------------------------------------------------------- MMA issuers
      const int x = warp - 1;
      auto kv_wait = [&](int e) -> bool {
        if (!wait_bar_w(bar(L::kKVFull + e % STAGES), (uint32_t)((e / STAGES) & 1), abort_flag,
                        status))
          return false;
        tc_fence_after();
        return true;
      };
      const uint64_t dq = desc_kmajor(sb + L::Q + (uint32_t)x * L::kTile);
      const uint64_t dkv_k = desc_kmajor(sb + L::KV);
      const uint64_t dkv_v = desc_mnmajor(sb + L::KV, 16384u);
      const int U = 2 * n;  // half-steps: u = 2j + h covers keys [64h, 64h + 64) of tile j
      auto qk = [&](int u) {
        const int j = u >> 1, h = u & 1;
        const uint64_t dk =
            desc_advance(dkv_k, (uint32_t)((2 * j) % STAGES) * L::kTile + (uint32_t)h * 8192u);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk >> 2) * 16384u + (uint32_t)(kk & 3) * 32u;
          mma_f16_ss_w(tmem + 128u * x + 64u * h, desc_advance(dq, off), desc_advance(dk, off),
                       kIdescQK, kk > 0 ? 1u : 0u);
        }
      };
      auto pv = [&](int u) {
        const int j = u >> 1, h = u & 1;
        const uint64_t dv = desc_advance(
            dkv_v, (uint32_t)((2 * j + 1) % STAGES) * L::kTile + (uint32_t)h * 8192u);
#pragma unroll
        for (int kk = 0; kk < kHalf / 16; ++kk)
          mma_f16_ts_w(tmem + 256u + 128u * x, tmem + 128u * x + 64u * h + 8u * kk,
                       desc_advance(dv, (uint32_t)kk * 2048u), kIdescPV,
                       (u > 0 || kk > 0) ? 1u : 0u);
      };
      bool ok = wait_bar_w(bar(L::kQFull), 0, abort_flag, status) && kv_wait(0);
      if (ok) {
        for (int h = 0; h < 2; ++h) {
          qk(h);
          tc_commit_w(bar(L::kSFull + 2 * x + h));
        }
        tc_commit_w(bar(L::kKVEmpty + 0));  // K_0 read by this tile
      }
      for (int u = 0; ok && u < U; ++u) {
        const int j = u >> 1, h = u & 1;
        const bool more = u + 2 < U;
        if (h == 0 && !(kv_wait(2 * j + 1) && (!more || kv_wait(2 * j + 2)))) break;
        if (!wait_bar_w(bar(L::kPFull + 2 * x + h), (uint32_t)((u >> 1) & 1), abort_flag, status))
          break;
        tc_fence_after();
        pv(u);
        tc_commit_w(bar(L::kPVDone + x));
        if (more) {  // into the slot PV(u) has just read (MMAs run in order)
          qk(u + 2);
          tc_commit_w(bar(L::kSFull + 2 * x + h));
        }
        if (h == 1) {
          tc_commit_w(bar(L::kKVEmpty + (2 * j + 1) % STAGES));
          if (more) tc_commit_w(bar(L::kKVEmpty + (2 * j + 2) % STAGES));
        }
      }
      tc_commit_w(bar(L::kOFull + x));
      tc_commit_w(bar(L::kDrain + x));
      wait_bar_drain(bar(L::kDrain + x), 0, status);
    }
  } else {
    regs_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int x = (warp - 4) >> 2;
    if (x < nx) {
      const int quarter = warp & 3;
      const int r = quarter * 32 + lane;
      const int64_t row = row0 + x * kTM + r;
      const bool live = row < geo.rows;
      const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
      const uint32_t t_sx = tmem + lane_base + 128u * x;
      const uint32_t t_o = tmem + lane_base + 256u + 128u * x;
      {  // gather this thread's query row; columns behind d and rows behind R are zero
        const int64_t per = (int64_t)geo.group * geo.n_q;
        const int64_t b = row / per, rem = row - b * per;
        const int64_t hg = rem / geo.n_q, i = rem - hg * geo.n_q;
        const T* src = q + b * geo.sb + (kvh * (int64_t)geo.group + hg) * geo.sh + i * geo.sn;
        const uint32_t tile = sb + L::Q + (uint32_t)x * L::kTile;
        uint4 w[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          w[c] = live && 8 * c < geo.d ? __ldg(reinterpret_cast<const uint4*>(src) + c)
                                       : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                           tile + (uint32_t)(c >> 3) * 16384u +
                           sw128_offset((uint32_t)r, 8u * (uint32_t)(c & 7))),
                       "r"(w[c].x), "r"(w[c].y), "r"(w[c].z), "r"(w[c].w)
                       : "memory");
        fence_proxy_async_smem();
        mbar_arrive(bar(L::kQFull));
      }
      const int U = 2 * n;
      float m_run = -INFINITY, l_run = 0.f;
      bool settled = false;  // warp-uniform: every row has a finite running maximum
      bool ok = true;
      for (int u = 0; u < U; ++u) {
        const int h = u & 1;
        const int64_t k0 = (int64_t)(t0 + (u >> 1)) * kTN + kHalf * h;
        const int left = (int)min((int64_t)kHalf, geo.P - k0);  // <= 0: nothing of this half
        ok = wait_bar_w(bar(L::kSFull + 2 * x + h), (uint32_t)((u >> 1) & 1), abort_flag, status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = t_sx + 64u * h;
        uint32_t sv[kHalf];
        tmem_ld32(t_s, sv);
        tmem_ld32(t_s + 32u, sv + 32);
        tmem_wait_ld();
        if (left < kHalf) {
#pragma unroll
          for (int c = 0; c < kHalf; ++c)
            if (c >= left) sv[c] = __float_as_uint(-INFINITY);
        }
        if (!settled) {
          float mx[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) mx[i] = __uint_as_float(sv[i]);
#pragma unroll
          for (int c = 8; c < kHalf; ++c) mx[c & 7] = fmaxf(mx[c & 7], __uint_as_float(sv[c]));
          const float rm = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                 fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
          if (m_run == -INFINITY) m_run = rm * scale_log2;
          settled = __all_sync(0xffffffffu, m_run != -INFINITY);
        }
        const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
        float mx[4];
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[kHalf / 2];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = -INFINITY;
        const float2 sc2 = make_float2(scale_log2, scale_log2);
        const float2 nm2 = make_float2(-m_use, -m_use);
#pragma unroll
        for (int i = 0; i < kHalf / 2; ++i) {
          const float s0 = __uint_as_float(sv[2 * i]), s1 = __uint_as_float(sv[2 * i + 1]);
          mx[i & 3] = max3f(mx[i & 3], s0, s1);
          const float2 x2 = __ffma2_rn(make_float2(s0, s1), sc2, nm2);
          const float2 p = make_float2(ex2(x2.x), ex2(x2.y));
          acc[i & 1] = __fadd2_rn(acc[i & 1], p);
          pk[i] = pack2<T>(p.x, p.y);  // to the input type: the MMA's A operand
        }
        const float rm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const float m_new = rm * scale_log2;
        const bool need = (m_run != -INFINITY) && (m_new > m_run + kRescaleLog2);
        float rsum = (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
        if (!__any_sync(0xffffffffu, need)) {
          tmem_st16(t_s, pk);
          tmem_st16(t_s + 16u, pk + 16);
        } else {
          ok = __all_sync(0xffffffffu,
                          u == 0 || wait_bar(bar(L::kPVDone + x), (uint32_t)((u - 1) & 1),
                                             abort_flag, status));
          if (!ok) break;
          tc_fence_after();
          const float alpha = need ? ex2(m_run - m_new) : 1.f;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t t[32];
            tmem_ld32(t_o + 32u * c, t);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) t[i] = __float_as_uint(__uint_as_float(t[i]) * alpha);
            tmem_st32(t_o + 32u * c, t);
          }
          if (need) {
            l_run *= alpha;
            m_run = m_new;
          }
          rsum = 0.f;
          const float m_re = (m_run == -INFINITY) ? 0.f : m_run;
#pragma unroll 1
          for (int c = 0; c < kHalf / 32; ++c) {
            uint32_t t[32], w[16];
            tmem_ld32(t_s + 32u * c, t);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float s0 = 32 * c + 2 * i < left ? __uint_as_float(t[2 * i]) : -INFINITY;
              const float s1 =
                  32 * c + 2 * i + 1 < left ? __uint_as_float(t[2 * i + 1]) : -INFINITY;
              const float p0 = ex2(fmaf(s0, scale_log2, -m_re));
              const float p1 = ex2(fmaf(s1, scale_log2, -m_re));
              rsum += p0 + p1;
              w[i] = pack2<T>(p0, p1);
            }
            tmem_st16(t_s + 16u * c, w);
          }
        }
        tmem_wait_st();
        l_run += rsum;
        tc_fence_before();
        mbar_arrive(bar(L::kPFull + 2 * x + h));
      }
      if (ok) ok = wait_bar_w(bar(L::kOFull + x), 0, abort_flag, status);
      if (ok) {
        tc_fence_after();
        const int64_t slot = ((int64_t)split * geo.kv_heads + kvh) * geo.rows + row;
        float* dst = part + slot * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t t[32];
          tmem_ld32(t_o + 32u * c, t);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(dst + 32 * c + 4 * i) =
                  make_uint4(t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]);
          }
        }
        if (live) stats[slot] = make_float2(m_run, l_run);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// merge
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 256;
enum OwnKind { kOwnNone = 0, kOwn16 = 1, kOwn32 = 2 };

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads)
    prefix_merge_kernel(const float* __restrict__ part, const float2* __restrict__ stats,
                        const void* __restrict__ own_o, const float* __restrict__ own_lse,
                        int own_kind, T* __restrict__ o, float* __restrict__ lse,
                        PrefixGeom geo) {
  constexpr int kLanes = D / 4;            // lanes per row, four columns each
  constexpr int kRows = kMergeThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t all = geo.rows * geo.kv_heads;
  const int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  if (at >= all) return;
  const int64_t kvh = at / geo.rows, row = at - kvh * geo.rows;
  const int64_t per = (int64_t)geo.group * geo.n_q;
  const int64_t b = row / per, rem = row - b * per;   // rem = head of the group * n_q + query
  const int64_t out = (b * geo.kv_heads + kvh) * per + rem;   // row of o [B, H, n_q]
  const bool on = lane * 4 < geo.d;
  const float own_l2 =
      own_kind == kOwnNone ? -INFINITY : own_lse[out] * kLog2e;   // log2 of the own weight
  float M = own_l2;
  for (int s = 0; s < geo.splits; ++s) M = fmaxf(M, stats[s * all + at].x);
  const float ref = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < geo.splits; ++s) {
    const float2 st = stats[s * all + at];
    const float f = ex2(st.x - ref);
    const float4 p = *reinterpret_cast<const float4*>(part + (s * all + at) * D + lane * 4);
    l += st.y * f;
    a.x += p.x * f;
    a.y += p.y * f;
    a.z += p.z * f;
    a.w += p.w * f;
  }
  if (own_kind != kOwnNone && on && own_l2 != -INFINITY) {
    const float f = ex2(own_l2 - ref);
    float4 p;
    if (own_kind == kOwn32) {
      p = *reinterpret_cast<const float4*>((const float*)own_o + out * geo.d + lane * 4);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>((const T*)own_o + out * geo.d + lane * 4);
      const T* e = reinterpret_cast<const T*>(&w);
      p = make_float4(Elem<T>::to(e[0]), Elem<T>::to(e[1]), Elem<T>::to(e[2]), Elem<T>::to(e[3]));
    }
    l += f;
    a.x += p.x * f;
    a.y += p.y * f;
    a.z += p.z * f;
    a.w += p.w * f;
  }
  if (!on) return;
  const float inv = 1.f / l;
  *reinterpret_cast<uint2*>(o + out * geo.d + lane * 4) =
      make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  if (lane == 0 && lse) lse[out] = (ref + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int tile_dim(int64_t d) {
  if (d <= 0 || d > 128 || d % 8 != 0) return 0;
  return d <= 64 ? 64 : 128;
}

// Key slices: whole waves of one CTA per SM, each as long as its tiles plus a set-up worth
// about three (Q gather, pipeline fill, epilogue), against the partial rows that every
// slice writes and the merge reads (a tile's time moves about 6 MB).
int prefix_splits(int64_t ctas, int n_tiles, int64_t part_bytes) {
  const int64_t sms = device_sm_count();
  int best = 1;
  double best_cost = 1e300;
  for (int ns = 1; ns <= std::min(n_tiles, 64); ++ns) {
    const int64_t waves = (ctas * ns + sms - 1) / sms;
    const double cost = (double)waves * ((n_tiles + ns - 1) / ns + 3) + ns * part_bytes / 3e6;
    if (cost < best_cost) {
      best_cost = cost;
      best = ns;
    }
  }
  return best;
}

bool prefix_geometry(int64_t B, int64_t H, int64_t kv_heads, int64_t n_q, int64_t P,
                     int64_t head_dim, PrefixGeom* geo) {
  if (B <= 0 || H <= 0 || n_q <= 0 || P <= 0 || P >= (1ll << 31) || tile_dim(head_dim) == 0)
    return false;
  if (kv_heads <= 0) kv_heads = H;
  if (H % kv_heads != 0 || kv_heads > 65535 || B >= (1ll << 31) || H >= (1ll << 31) ||
      n_q >= (1ll << 31))
    return false;
  const int64_t group = H / kv_heads;
  if (B * group >= (1ll << 31) || B * group * n_q >= (1ll << 38)) return false;
  geo->rows = B * group * n_q;
  geo->P = P;
  geo->group = (int)group;
  geo->n_q = (int)n_q;
  geo->kv_heads = (int)kv_heads;
  geo->d = (int)head_dim;
  geo->n_tiles = ceil_div_i(P, kTN);
  const int64_t pairs = (geo->rows + kPair * kTM - 1) / (kPair * kTM);
  geo->splits = prefix_splits(pairs * kv_heads, geo->n_tiles,
                              geo->rows * kv_heads * tile_dim(head_dim) * 4);
  return true;
}

int64_t stats_bytes(const PrefixGeom& g) {
  return (g.splits * g.kv_heads * g.rows * (int64_t)sizeof(float2) + 255) / 256 * 256;
}
int64_t part_bytes(const PrefixGeom& g) {
  return g.splits * g.kv_heads * g.rows * (int64_t)tile_dim(g.d) * (int64_t)sizeof(float);
}

template <typename T, int D, int STAGES>
int launch_prefix(const void* q, const void* k, const void* v, const void* own_o,
                  const float* own_lse, int own_kind, void* o, float* lse, float scale,
                  const PrefixGeom& geo, void* ws, cudaStream_t s) {
  using L = PrefixLayout<D, STAGES>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mk, mv;
  const Strides3 st{geo.kv_heads * geo.P * geo.d, geo.P * geo.d, geo.d};
  if (int rc = make_tmap_4d(&mk, k, kBF16, (uint64_t)geo.d, (uint64_t)geo.P,
                            (uint64_t)geo.kv_heads, 1, st, kTN))
    return rc;
  if (int rc = make_tmap_4d(&mv, v, kBF16, (uint64_t)geo.d, (uint64_t)geo.P,
                            (uint64_t)geo.kv_heads, 1, st, kTN))
    return rc;
  float2* stats = (float2*)ws;
  float* part = (float*)((char*)ws + stats_bytes(geo));
  auto kern = prefix_tc_kernel<T, D, STAGES>;
  if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)L::kAlloc),
                          "cudaFuncSetAttribute(prefix_tc)"))
    return rc;
  const int64_t pairs = (geo.rows + kPair * kTM - 1) / (kPair * kTM);
  if (pairs >= (1ll << 31)) return fail(SBFA_ERR_UNSUPPORTED, "prefix: too many query rows");
  {
    LaunchScope ls("prefix_tc_kernel", s);
    kern<<<dim3((unsigned)pairs, (unsigned)geo.kv_heads, (unsigned)geo.splits), kThreads,
           L::kAlloc, s>>>((const T*)q, mk, mv, part, stats, scale * kLog2e, geo,
                           device_status_ptr());
  }
  if (int rc = check_launch("prefix_tc_kernel")) return rc;
  const int64_t rows_per = kMergeThreads / (D / 4);
  const int64_t blocks = (geo.rows * geo.kv_heads + rows_per - 1) / rows_per;
  if (blocks >= (1ll << 31)) return fail(SBFA_ERR_UNSUPPORTED, "prefix: too many query rows");
  {
    LaunchScope ls("prefix_merge_kernel", s);
    prefix_merge_kernel<T, D><<<(unsigned)blocks, kMergeThreads, 0, s>>>(
        part, stats, own_o, own_lse, own_kind, (T*)o, lse, geo);
  }
  return check_launch("prefix_merge_kernel");
}

}  // namespace
}  // namespace sbfa

using namespace sbfa;

extern "C" int64_t sbfa_prefix_workspace_bytes(int64_t B, int64_t H, int64_t kv_heads,
                                               int64_t n_q, int64_t P, int64_t head_dim) {
  PrefixGeom geo;
  if (!prefix_geometry(B, H, kv_heads, n_q, P, head_dim, &geo)) return 0;
  return stats_bytes(geo) + part_bytes(geo);
}

extern "C" int sbfa_prefix_attend(const void* q, const int64_t* q_strides, const void* k_prefix,
                                  const void* v_prefix, const void* own_o, const float* own_lse,
                                  int own_kind, void* o, float* lse, int64_t B, int64_t H,
                                  int64_t kv_heads, int64_t n_q, int64_t P, int64_t head_dim,
                                  int dtype, double softmax_scale, void* ws, int64_t ws_bytes,
                                  void* stream) {
  if (dtype != SBFA_F16 && dtype != SBFA_BF16)
    return fail(SBFA_ERR_UNSUPPORTED, "sbfa_prefix_attend: dtype must be float16 or bfloat16");
  if (tile_dim(head_dim) == 0)
    return fail(SBFA_ERR_UNSUPPORTED,
                "sbfa_prefix_attend: head_dim must be a multiple of 8 and at most 128");
  PrefixGeom geo;
  if (!prefix_geometry(B, H, kv_heads, n_q, P, head_dim, &geo))
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_attend: sizes must be positive and below 2^31, H "
                                  "a multiple of kv_heads");
  if (!(softmax_scale > 0) || softmax_scale > 1e30)
    return fail(SBFA_ERR_INVALID, "softmax_scale must be positive and finite");
  if (!q || !k_prefix || !v_prefix || !o)
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_attend: NULL tensor pointer");
  if (own_kind < 0 || own_kind > 2 || (own_kind != 0 && (!own_o || !own_lse)))
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_attend: own_o and own_lse must match own_kind");
  geo.sn = q_strides ? q_strides[2] : head_dim;
  geo.sh = q_strides ? q_strides[1] : n_q * head_dim;
  geo.sb = q_strides ? q_strides[0] : H * n_q * head_dim;
  if (geo.sb < 0 || geo.sh < 0 || geo.sn < 0 || geo.sb % 8 || geo.sh % 8 || geo.sn % 8)
    return fail(SBFA_ERR_INVALID,
                "sbfa_prefix_attend: q strides must be non-negative multiples of 8 elements");
  for (const void* p : {q, k_prefix, v_prefix, own_o, (const void*)o, (const void*)ws})
    if ((uintptr_t)p & 15u)
      return fail(SBFA_ERR_INVALID, "sbfa_prefix_attend: tensors must be 16-byte aligned");
  const int64_t need = stats_bytes(geo) + part_bytes(geo);
  if (ws == nullptr || ws_bytes < need)
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_attend: workspace too small (need " +
                                      std::to_string(need) + " bytes)");
  cudaStream_t s = (cudaStream_t)stream;
  const float sc = (float)softmax_scale;
#define SBFA_PREFIX(TT, DD, ST) \
  return launch_prefix<TT, DD, ST>(q, k_prefix, v_prefix, own_o, own_lse, own_kind, o, lse, sc, \
                                   geo, ws, s)
  if (tile_dim(head_dim) == 64) {
    if (dtype == SBFA_BF16) SBFA_PREFIX(__nv_bfloat16, 64, 8);
    SBFA_PREFIX(__half, 64, 8);
  }
  if (dtype == SBFA_BF16) SBFA_PREFIX(__nv_bfloat16, 128, 5);
  SBFA_PREFIX(__half, 128, 5);
#undef SBFA_PREFIX
}
