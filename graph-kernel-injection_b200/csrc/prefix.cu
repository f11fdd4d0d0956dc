// Attention of a batch to a prefix that all its sequences share.
//
// Every query sees every prefix token, so the n_q query rows of all B sequences and
// of the G query heads of a key/value head form one matrix of R = B G n_q rows per
// key/value head: O_p = softmax(scale Q K^T) V with K, V read once for the batch
// instead of once per sequence.  Row r is (sequence, head of the group, query) =
// (r / (G n_q), r / n_q % G, r % n_q).
//
// prefix_tc_kernel: one CTA per (256 rows, key/value head) or per slice of its keys, the
// pipeline of the block-sparse forward: a TMA warp streams K and V tiles of 128 keys
// through a ring, one warp per 128-row tile issues the MMAs, a warpgroup per tile
// runs the online softmax on TMEM (see attn_tc.cu for the TMEM plan).  Q rows come from
// scattered places, so the softmax threads gather them (a thread per row) into the
// swizzled operand tile.  With 128 rows or fewer in the CTA the second tile's
// warps leave at once.  The floor of few rows against a long prefix is HBM (4 D bytes per
// key), of many the tensor cores (4 D operations per row and key); what holds either is the latency
// of a tile's score / weight / PV chain (8 x 512 prompt tokens of 32 heads behind 8192 shared ones
// 505 us, 0.67 of the measured burst rate).
//
// Weights are rounded to the input type, the MMA's operand, before PV; their sum l is not.  With
// bf16 that is the larger part of the error against 64 bits: 2.0e-3 of O in decode, 2.3e-3 in
// prompts, where rounding O alone leaves 1.7e-3.
//
// The batch's own prompts (n_q tokens each, causal window and own sinks) follow as more key
// tiles of the same pass: a tile of 128 keys of one sequence, or of 128 / 2^k short
// sequences with 2^k >= n_q rows each, in which each query row sees one interval
// of columns, or two where a tile holds sinks.  So a prompt takes one launch, and its two parts share one softmax and
// one rounding.  A value row in a tile belongs to some of the tile's query rows only, and a
// weight of zero does not keep a NaN or an infinity out of the others' sums: a fourth
// warp looks over every own V tile as it arrives, replaces such elements by zeros and
// has the epilogue add them to the rows that do see them.
//
// Slices.  Whole waves of CTAs take all keys of their rows and write O themselves.  The
// rest (all of them in a decode step) would leave most SMs idle, so their keys are cut
// into slices, which leave fp32 rows with (m, l) that prefix_merge_kernel joins.  Either
// epilogue also joins the row's attention over its own tokens that a cache's kernel
// has computed (already normalised, with its log-sum-exp).
//
// A decode step behind a prefix is bound by that chain here (alone, before 32768 tokens, no unit is
// busy for more than half of the time: tensor 39 %, MUFU 39 %, DRAM 35 %) and by HBM in the 8-bit
// cache's kernel, so the two share the GPU: this kernel takes fewer SMs with longer slices, the
// cache's kernel starts at once on the others and on those that come free, and the merge waits for
// both (64 sequences, 32 heads over 8, 16384 shared tokens and ragged rings of 1024: 56 us one
// after the other, 49 us so; 16 sequences behind 8192: 35 and 23).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "quant_cache.cuh"
#include "tc_attn_common.cuh"

namespace sbfa {
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
  int64_t sb, sh, sn;  // q strides (batch, head, query)
  int rows;            // R, rows per key/value head (below 2^31 - 256)
  int P;
  int group, n_q, kv_heads, batch, d;
  int pairs;           // 256-row tiles per key/value head
  int n_full, n_tail;  // units (tile, head) that take all keys / that are cut into slices
  int splits;          // slices of a tail unit
  int n_tiles;         // 128-key tiles of the prefix
  int own;             // whether own tokens follow the prefix
  int window, box;     // their window; rows of a TMA box of own keys (128 / box sequences a tile)
  int sink;            // first own tokens that every later one sees
};

// How a row's attention to its own tokens comes from a cache's kernel: O of the output type (every
// row saw a key), or fp32 with LSE -inf for a row that saw none.
enum OwnKind { kOwnNone = 0, kOwn16 = 1, kOwn32 = 2 };

// Where O goes and what a cache's kernel contributes to it.
struct PrefixOut {
  void* o;               // [B, H, n_q, d]
  float* lse;            // [B, H, n_q] or NULL
  const void* own_o;
  const float* own_lse;
  int own_kind;
  const void* own_v;     // own value rows and their strides (prompts)
  Strides3 sv;
  float* part;           // [splits][n_tail * 256][D]
  float2* stats;         // [splits][n_tail * 256] (m, l)
};

// Row of O for row `row` of a key/value head.
__device__ __forceinline__ int64_t out_row(const PrefixGeom& g, int kvh, int row) {
  const int per = g.group * g.n_q;
  const int b = row / per;
  return ((int64_t)b * g.kv_heads + kvh) * per + (row - b * per);
}

// The own-key tiles that rows [row0, row1) need, in order: sequence by sequence (box == 128;
// the first one's with its sinks and from its window's oldest key), or blocks of 128 / box sequences.
struct OwnTiles {
  int b0, kt0, c0;   // first sequence (or block), its window's first tile, its tiles in all
  int sinks;         // of them ahead of the window's
  int full;          // tiles of a whole sequence
  int count;
  __device__ __forceinline__ OwnTiles(const PrefixGeom& g, int row0, int row1) {
    b0 = kt0 = c0 = sinks = count = 0;
    full = 1;
    if (!g.own) return;
    const int per = g.group * g.n_q;
    b0 = row0 / per;
    const int b1 = (row1 - 1) / per;
    if (g.box < kTN) {
      const int seqs = kTN / g.box;
      b0 /= seqs;
      c0 = 1;
      count = b1 / seqs - b0 + 1;
      return;
    }
    full = (g.n_q + kTN - 1) / kTN;
    // queries [q_lo, q_hi] of a run of rows: of several heads, all of them
    const int lo = row0 - b0 * per, hi = min(row1 - b0 * per, per) - 1;
    const bool one = lo / g.n_q == hi / g.n_q;
    const int q_lo = one ? lo % g.n_q : 0, q_hi = one ? hi % g.n_q : g.n_q - 1;
    kt0 = max(0, q_lo - g.window + 1) / kTN;
    sinks = min(kt0, (g.sink + kTN - 1) / kTN);
    c0 = sinks + q_hi / kTN - kt0 + 1;
    count = c0;
    if (b1 > b0) {
      const int last = row1 - 1 - b1 * per;
      count += (b1 - b0 - 1) * full + (last < g.n_q ? last : g.n_q - 1) / kTN + 1;
    }
  }
  // own tile u: sequence (or block of them) and its key tile
  __device__ __forceinline__ void at(int u, int* b, int* kt) const {
    if (u < c0) {
      *b = b0;
      *kt = u < sinks ? u : kt0 + u - sinks;
    } else {
      *b = b0 + 1 + (u - c0) / full;
      *kt = (u - c0) % full;
    }
  }
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
  static constexpr int kVRaw = 15 + 2 * STAGES;   // [STAGES] an own V tile has arrived
  static constexpr int kNumBars = 15 + 3 * STAGES;
  static constexpr uint32_t MISC = BAR + kNumBars * 8;  // TMEM base, abort flag, bad V flag
  static constexpr uint32_t kAlloc = MISC + 16 + 1024;
  // key tiles from one own V tile to the next in the same ring slot
  static constexpr int kVPeriod = STAGES % 2 ? STAGES : STAGES / 2;
};

template <typename T, int D, int STAGES>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tc_kernel(const T* __restrict__ q, const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv,
                     const __grid_constant__ CUtensorMap tmok,
                     const __grid_constant__ CUtensorMap tmov, PrefixOut out, float scale_log2,
                     PrefixGeom geo, int* status) {
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
  volatile int* bad_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 8);

  griddep_launch();   // the cache's kernel or the merge may take what SMs are left
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bid = (int)blockIdx.x;
  const bool sliced = bid >= geo.n_full;
  const int tail = sliced ? (bid - geo.n_full) % geo.n_tail : 0;
  const int split = sliced ? (bid - geo.n_full) / geo.n_tail : 0;
  const int splits = sliced ? geo.splits : 1;
  const int unit = sliced ? geo.n_full + tail : bid;
  const int kvh = unit / geo.pairs;
  const int row0 = unit % geo.pairs * (kPair * kTM);
  const int nx = row0 + kTM < geo.rows ? 2 : 1;  // tiles with rows in them
  const OwnTiles own(geo, row0, min(row0 + kPair * kTM, geo.rows));
  const int n_all = geo.n_tiles + (geo.own ? own.count : 0);
  // slices of n_all / splits tiles, none empty (splits <= n_tiles)
  const int t0 = (int)((int64_t)split * n_all / splits);
  const int n = (int)((int64_t)(split + 1) * n_all / splits) - t0;
  const int j_own = max(0, geo.n_tiles - t0);   // the first of them with own keys (n if none)

  // phase of kVRaw in which own tile j arrives: how often its slot has held an own V before
  auto own_phase = [&](int j) { return (uint32_t)(((j - j_own) / L::kVPeriod) & 1); };
  // K (part 0) or V (part 1) of key tile t into ring slot s.  Own V tiles complete on kVRaw, and
  // the warp that looks them over completes kKVFull.
  auto load_tile = [&](int t, int part, int s) {
    const uint32_t dst = sb + L::KV + (uint32_t)s * L::kTile;
    const uint32_t full = bar((part == 1 && t >= geo.n_tiles ? L::kVRaw : L::kKVFull) + s);
    mbar_expect_tx(full, L::kTile);
    if (t < geo.n_tiles) {
      for (int r = 0; r < kBoxes; ++r)
        tma_load_4d(dst + r * 16384u, part == 0 ? &tmk : &tmv, full, 64 * r, t * kTN, kvh, 0);
      return;
    }
    int b, kt;
    own.at(t - geo.n_tiles, &b, &kt);
    const int seqs = kTN / geo.box;
    for (int i = 0; i < seqs; ++i)   // a sequence behind the last one reads as zeros
      for (int r = 0; r < kBoxes; ++r)
        tma_load_4d(dst + r * 16384u + (uint32_t)(i * geo.box) * 128u,
                    part == 0 ? &tmok : &tmov, full, 64 * r, kt * kTN, kvh, b * seqs + i);
  };

  if (threadIdx.x == 0) {
    mbar_init(bar(L::kQFull), 128 * nx);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar(L::kKVFull + s), 1);
      mbar_init(bar(L::kKVEmpty + s), nx);
      mbar_init(bar(L::kVRaw + s), 1);
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
    *bad_flag = 0;
    mbar_init_fence();
    // the first K and V on their way before the TMEM allocation and the CTA-wide sync
    load_tile(t0, 0, 0);
    load_tile(t0, 1, 1);
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
          load_tile(t0 + j, part_, s);
          issued = e + 1;
        }
      }
      for (int s = 0; s < STAGES; ++s) {  // our own copies still in flight
        if (issued <= s) continue;
        const int e = s + (issued - 1 - s) / STAGES * STAGES;   // the slot's last entry
        if (e % 2 && e / 2 >= j_own)
          wait_bar_drain(bar(L::kVRaw + s), own_phase(e / 2), status);
        else
          wait_bar_drain(bar(L::kKVFull + s), (uint32_t)((e / STAGES) & 1), status);
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
    } else if (warp == 3) {
      // ---------------------------------------------------------- own V tiles
      constexpr uint32_t kInf = kBF16 ? 0x7f80u : 0x7c00u;   // 16 bits of infinity
      for (int j = j_own; j < n; ++j) {
        const int e = 2 * j + 1, s = e % STAGES;
        if (!wait_bar_w(bar(L::kVRaw + s), own_phase(j), abort_flag, status)) break;
        const uint32_t tile = sb + L::KV + (uint32_t)s * L::kTile + 16u * (uint32_t)lane;
        bool bad = false;
#pragma unroll 8
        for (uint32_t off = 0; off < L::kTile; off += 512u) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(tile + off));
          const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                      __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
          bad |= (m & 0xffffu) >= kInf || (m >> 16) >= kInf;
        }
        if (__any_sync(0xffffffffu, bad)) {   // rare: zeros in the place of such elements
          for (uint32_t off = 0; off < L::kTile; off += 512u)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
              uint32_t w;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(tile + off + 4u * i));
              if ((w & 0x7fffu) >= kInf) w &= 0xffff0000u;
              if ((w >> 16 & 0x7fffu) >= kInf) w &= 0xffffu;
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(tile + off + 4u * i), "r"(w) : "memory");
            }
          *bad_flag = 1;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::kKVFull + s));
      }
    }
  } else {
    regs_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int x = (warp - 4) >> 2;
    if (x < nx) {
      const int quarter = warp & 3;
      const int r = quarter * 32 + lane;
      const int row = row0 + x * kTM + r;
      const bool live = row < geo.rows;
      const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
      const uint32_t t_sx = tmem + lane_base + 128u * x;
      const uint32_t t_o = tmem + lane_base + 256u + 128u * x;
      const int per = geo.group * geo.n_q;
      const int seq = row / per;
      const int hg = (row - seq * per) / geo.n_q;
      const int iq = row - seq * per - hg * geo.n_q;   // the row's query of its sequence
      // Columns of own key tile t that this row sees: [lo, hi), and from off, its sequence's token
      // 0, to off + sink as far as they lie ahead of hi.  None in a tile of other sequences.
      auto own_keys = [&](int t, int* lo, int* hi, int* off) {
        int b, kt;
        own.at(t - geo.n_tiles, &b, &kt);
        const int seqs = kTN / geo.box;
        const int s = seq - b * seqs;                  // this row's sequence in the tile
        *off = s * geo.box - kt * kTN;
        *lo = *off + max(iq - geo.window + 1, 0);
        *hi = live && s >= 0 && s < seqs ? *off + iq + 1 : 0;
      };
      {  // gather this warp's query rows, D / 8 lanes a row; columns behind d and rows behind
         // R are zero.  (A row per lane would touch 32 lines with every load: 1.5 us more.)
        const T* mine = live ? q + seq * geo.sb + ((int64_t)kvh * geo.group + hg) * geo.sh +
                                   iq * geo.sn
                             : nullptr;
        const uint32_t tile = sb + L::Q + (uint32_t)x * L::kTile;
        constexpr int kChunks = D / 8;
        uint4 w[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const int rr = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
          const T* src = (const T*)__shfl_sync(0xffffffffu, (unsigned long long)mine, rr);
          w[i] = src != nullptr && 8 * c < geo.d ? __ldg(reinterpret_cast<const uint4*>(src) + c)
                                                 : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const int rr = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                           tile + (uint32_t)(c >> 3) * 16384u +
                           sw128_offset((uint32_t)(quarter * 32 + rr), 8u * (uint32_t)(c & 7))),
                       "r"(w[i].x), "r"(w[i].y), "r"(w[i].z), "r"(w[i].w)
                       : "memory");
        }
        fence_proxy_async_smem();
        mbar_arrive(bar(L::kQFull));
      }
      const int U = 2 * n;
      float m_run = -INFINITY, l_run = 0.f;
      bool settled = false;  // warp-uniform: every row has a finite running maximum
      bool ok = true;
      for (int u = 0; u < U; ++u) {
        const int h = u & 1;
        const int t = t0 + (u >> 1);
        // visible keys of this half-step: one interval of columns
        uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
        bool all_vis = t < geo.n_tiles - 1;   // all but the prefix's last tile are full
        if (!all_vis) {
          int lo = 0, hi, off;
          if (t < geo.n_tiles)
            hi = geo.P - t * kTN;
          else
            own_keys(t, &lo, &hi, &off);
          vis[0] = range_bits(lo, hi, kHalf * h);
          vis[1] = range_bits(lo, hi, kHalf * h + 32);
          if (t >= geo.n_tiles && geo.sink > 0) {
            const int end = min(off + geo.sink, hi);
            vis[0] |= range_bits(off, end, kHalf * h);
            vis[1] |= range_bits(off, end, kHalf * h + 32);
          }
          all_vis = __all_sync(0xffffffffu, (vis[0] & vis[1]) == 0xffffffffu);
        }
        ok = wait_bar_w(bar(L::kSFull + 2 * x + h), (uint32_t)((u >> 1) & 1), abort_flag, status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = t_sx + 64u * h;
        uint32_t sv[kHalf];
        tmem_ld32(t_s, sv);
        tmem_ld32(t_s + 32u, sv + 32);
        tmem_wait_ld();
        if (!all_vis) {
#pragma unroll
          for (int c = 0; c < kHalf; ++c)
            if (!((vis[c >> 5] >> (c & 31)) & 1u)) sv[c] = __float_as_uint(-INFINITY);
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
            uint32_t ov[32];
            tmem_ld32(t_o + 32u * c, ov);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st32(t_o + 32u * c, ov);
          }
          if (need) {
            l_run *= alpha;
            m_run = m_new;
          }
          rsum = 0.f;
          const float m_re = (m_run == -INFINITY) ? 0.f : m_run;
#pragma unroll 1
          for (int c = 0; c < kHalf / 32; ++c) {
            uint32_t sc[32], w[16];
            tmem_ld32(t_s + 32u * c, sc);
            tmem_wait_ld();
            const uint32_t vb = c == 0 ? vis[0] : vis[1];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float s0 = ((vb >> (2 * i)) & 1u) ? __uint_as_float(sc[2 * i]) : -INFINITY;
              const float s1 =
                  ((vb >> (2 * i + 1)) & 1u) ? __uint_as_float(sc[2 * i + 1]) : -INFINITY;
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
        // A row's 2 D bytes pass through this warp's part of the Q tile, which is no
        // longer read, so that a row is written by adjacent lanes.
        const uint32_t stage = sb + L::Q + (uint32_t)x * L::kTile;
        constexpr int kChunks = D / 8;
        auto put = [&](int c, uint32_t a, uint32_t b, uint32_t e, uint32_t f) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                           stage + (uint32_t)(c >> 3) * 16384u +
                           sw128_offset((uint32_t)r, 8u * (uint32_t)(c & 7))),
                       "r"(a), "r"(b), "r"(e), "r"(f)
                       : "memory");
        };
        auto flush = [&](char* dst, int chunks) {   // chunks of 16 bytes that exist
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int rr = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
            char* to = (char*)__shfl_sync(0xffffffffu, (unsigned long long)dst, rr);
            uint4 w;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                         : "r"(stage + (uint32_t)(c >> 3) * 16384u +
                               sw128_offset((uint32_t)(quarter * 32 + rr), 8u * (uint32_t)(c & 7))));
            if (to != nullptr && c < chunks) reinterpret_cast<uint4*>(to)[c] = w;
          }
          __syncwarp();
        };
        // columns [c0, c0 + 32) of what the fourth warp took out of the value rows that this row
        // sees in this CTA's own tiles (another slice adds its own: here such a row may have no key
        // at all, and then a weight of 0 in the merge, which an infinity must not meet)
        const bool patch = live && *bad_flag != 0;
        auto put_back = [&](float* f, int c0) {
          const T* v = (const T*)out.own_v + seq * out.sv.b + (int64_t)kvh * out.sv.h + c0;
          for (int j = j_own; j < n; ++j) {
            int lo, hi, off;
            own_keys(t0 + j, &lo, &hi, &off);
            for (int c = max(off, 0); c < min(hi, kTN); ++c) {
              if (c >= off + geo.sink && c < lo) continue;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c0 + i < geo.d) {
                  const float y = Elem<T>::to(v[(c - off) * out.sv.n + i]);
                  if (!(fabsf(y) < INFINITY)) f[i] += y;
                }
            }
          }
        };
        if (sliced) {
          const int64_t all = (int64_t)geo.n_tail * (kPair * kTM);
          const int64_t slot = split * all + (int64_t)tail * (kPair * kTM) + x * kTM + r;
          if (live) out.stats[slot] = make_float2(m_run, l_run);
#pragma unroll
          for (int half = 0; half < 2; ++half) {   // D / 2 fp32 columns at a time
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              uint32_t ov[32];
              tmem_ld32(t_o + (uint32_t)(half * (D / 2) + 32 * c), ov);
              tmem_wait_ld();
              if (patch) put_back(reinterpret_cast<float*>(ov), half * (D / 2) + 32 * c);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                put(8 * c + i, ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
            }
            flush(live ? (char*)(out.part + slot * D + half * (D / 2)) : nullptr, kChunks);
          }
        } else {
          const int64_t at = live ? out_row(geo, kvh, row) : 0;
          const float own_l2 =
              out.own_kind != kOwnNone && live ? out.own_lse[at] * kLog2e : -INFINITY;
          const float M = fmaxf(m_run, own_l2);
          const float f_own = own_l2 == -INFINITY ? 0.f : ex2(own_l2 - M);
          const float f_pre = ex2(m_run - M);
          const float l = l_run * f_pre + f_own;
          const float inv = 1.f / l;
          const float w_pre = f_pre * inv, w_own = f_own * inv;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t ov[32];
            tmem_ld32(t_o + 32u * c, ov);
            tmem_wait_ld();
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(ov[i]) * w_pre;
            if (patch) put_back(f, 32 * c);
            if (f_own != 0.f) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (32 * c + i < geo.d)
                  f[i] += w_own * Elem<T>::to(((const T*)out.own_o)[at * geo.d + 32 * c + i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              put(4 * c + i, pack2<T>(f[8 * i], f[8 * i + 1]), pack2<T>(f[8 * i + 2], f[8 * i + 3]),
                  pack2<T>(f[8 * i + 4], f[8 * i + 5]), pack2<T>(f[8 * i + 6], f[8 * i + 7]));
          }
          flush(live ? (char*)((T*)out.o + at * geo.d) : nullptr, geo.d / 8);
          if (live && out.lse) out.lse[at] = (M + log2f(l)) * kLn2;
        }
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

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads)
    prefix_merge_kernel(PrefixOut po, PrefixGeom geo) {
  constexpr int kLanes = D / 4;            // lanes per row, four columns each
  constexpr int kRows = kMergeThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t all = (int64_t)geo.n_tail * (kPair * kTM);
  const int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  const int unit = geo.n_full + (int)(at / (kPair * kTM));
  const int row = unit % geo.pairs * (kPair * kTM) + (int)(at % (kPair * kTM));
  griddep_wait();
  const bool live = at < all && row < geo.rows;   // uniform over a row's lanes
  const int64_t out = live ? out_row(geo, unit / geo.pairs, row) : 0;
  const bool on = lane * 4 < geo.d;
  const float own_l2 = live && po.own_kind != kOwnNone ? po.own_lse[out] * kLog2e : -INFINITY;
  // the first slices' columns are under way while the weights are worked out
  constexpr int kAhead = 8;
  const float* src = po.part + (live ? at : 0) * D + lane * 4;
  float4 p[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    p[j] = live && j < geo.splits ? *reinterpret_cast<const float4*>(src + j * all * D)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
  // every slice's m and l at once, a lane each (at most 64 slices, 16 or 32 lanes)
  float2 st[64 / kLanes];
  float M = own_l2;
#pragma unroll
  for (int i = 0; i < 64 / kLanes; ++i) {
    const int s = i * kLanes + lane;
    st[i] = live && s < geo.splits ? po.stats[s * all + at] : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, st[i].x);
  }
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const float ref = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  float w[64 / kLanes];
#pragma unroll
  for (int i = 0; i < 64 / kLanes; ++i) {
    w[i] = ex2(st[i].x - ref);
    l += st[i].y * w[i];
  }
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float f_own = own_l2 == -INFINITY ? 0.f : ex2(own_l2 - ref);
  l += f_own;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float4 p, float f) {
    a.x += p.x * f;
    a.y += p.y * f;
    a.z += p.z * f;
    a.w += p.w * f;
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j)   // a slice that is not there has weight 0 and zero columns
    add(p[j], __shfl_sync(0xffffffffu, w[0], j, kLanes));
#pragma unroll
  for (int i = 0; i < 64 / kLanes; ++i)
#pragma unroll 8
    for (int j = i == 0 ? kAhead : 0; j < kLanes; ++j) {
      if (i * kLanes + j >= geo.splits) break;
      add(*reinterpret_cast<const float4*>(src + (i * kLanes + j) * all * D),
          __shfl_sync(0xffffffffu, w[i], j, kLanes));
    }
  if (!live || !on) return;
  if (f_own != 0.f) {
    float4 p;
    if (po.own_kind == kOwn32) {
      p = *reinterpret_cast<const float4*>((const float*)po.own_o + out * geo.d + lane * 4);
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>((const T*)po.own_o + out * geo.d + lane * 4);
      const T* e = reinterpret_cast<const T*>(&x);
      p = make_float4(Elem<T>::to(e[0]), Elem<T>::to(e[1]), Elem<T>::to(e[2]), Elem<T>::to(e[3]));
    }
    add(p, f_own);
  }
  const float inv = 1.f / l;
  *reinterpret_cast<uint2*>((T*)po.o + out * geo.d + lane * 4) =
      make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  if (lane == 0 && po.lse) po.lse[out] = (ref + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int tile_dim(int64_t d) {
  if (d <= 0 || d > 128 || d % 8 != 0) return 0;
  return d <= 64 ? 64 : 128;
}

// Slices of the tail units, by the time that they take in us: whole waves of one CTA per SM, each
// as long as its tiles (2.15 us for two query tiles, 1.5 for one) plus 6 us (Q gather, pipeline
// fill, epilogue), and the partial rows that every slice writes and the merge reads back (3 MB
// a us; half as dear with the waves of fewer, longer slices beside another kernel).
// beside: SM time that a kernel running beside this one needs; it fills what SMs this one leaves.
int prefix_splits(int64_t units, int n_tiles, bool two, int64_t part_bytes, double beside) {
  const int64_t sms = device_sm_count();
  const double tile = two ? 2.15 : 1.5, per_us = beside > 0 ? 6e6 : 3e6;
  int best = 1;
  double best_cost = 1e300;
  for (int ns = 1; ns <= std::min(n_tiles, 64); ++ns) {
    const int64_t waves = (units * ns + sms - 1) / sms;
    const double cta = (n_tiles + ns - 1) / ns * tile + 6;
    const double busy = (beside + units * ns * cta) / sms;
    const double cost = std::max(waves * cta, busy) + (ns > 1 ? ns * part_bytes / per_us + 4 : 0);
    if (cost < best_cost) {
      best_cost = cost;
      best = ns;
    }
  }
  return best;
}

bool prefix_geometry(int64_t B, int64_t H, int64_t kv_heads, int64_t n_q, int64_t P,
                     int64_t head_dim, int64_t window, PrefixGeom* geo,
                     const sbfa_qcache* cache = nullptr) {
  if (B <= 0 || H <= 0 || n_q <= 0 || P <= 0 || P >= (1ll << 31) - kTN || window < 0 ||
      tile_dim(head_dim) == 0)
    return false;
  if (kv_heads <= 0) kv_heads = H;
  if (H % kv_heads != 0 || B >= (1ll << 31) || H >= (1ll << 31) || n_q >= (1ll << 30))
    return false;
  const int64_t group = H / kv_heads;
  // rows of a key/value head, and CTAs, in 31 bits
  if (B * group >= (1ll << 31) || B * group * n_q >= (1ll << 31) - 512) return false;
  geo->rows = (int)(B * group * n_q);
  const int64_t pairs = ((int64_t)geo->rows + kPair * kTM - 1) / (kPair * kTM);
  const int64_t units = pairs * kv_heads;
  if (units >= (1ll << 30)) return false;
  geo->sb = geo->sh = geo->sn = 0;
  geo->P = (int)P;
  geo->group = (int)group;
  geo->n_q = (int)n_q;
  geo->kv_heads = (int)kv_heads;
  geo->batch = (int)B;
  geo->d = (int)head_dim;
  geo->pairs = (int)pairs;
  geo->n_tiles = ceil_div_i(P, kTN);
  geo->own = window > 0;
  geo->window = (int)std::min<int64_t>(window, n_q);
  geo->sink = 0;
  // a box of own keys holds one sequence's rows: the least power of two, at least the 8 rows
  // of a swizzle atom; more than 64 rows take whole tiles of one sequence
  int box = 8;
  while (box < n_q && box < kTN) box *= 2;
  geo->box = box;
  const int64_t unit_bytes = (int64_t)kPair * kTM * tile_dim(head_dim) * 4;
  const bool two = geo->rows > kTM;
  if (cache != nullptr) {
    // beside the cache's kernel, which reads a full cache at about 30 GB/s per SM, its ramps and
    // last wave counted; its result is joined by the merge, so every unit leaves partial rows
    const double beside = 2.0 * B * kv_heads * (double)(cache->sink + cache->window) *
                          (double)(head_dim + 1) / 30e3;
    geo->n_full = 0;
    geo->n_tail = (int)units;
    geo->splits = prefix_splits(units, geo->n_tiles, two, units * unit_bytes, beside);
    return true;
  }
  const int sms = device_sm_count();
  geo->n_full = (int)(units / sms * sms);
  geo->n_tail = (int)(units - geo->n_full);
  geo->splits = 1;
  if (geo->n_tail > 0)
    geo->splits = prefix_splits(geo->n_tail, geo->n_tiles, two, geo->n_tail * unit_bytes, 0);
  if (geo->splits == 1) {  // nothing to cut
    geo->n_full += geo->n_tail;
    geo->n_tail = 0;
  }
  return true;
}

int64_t tail_rows(const PrefixGeom& g) {
  return (int64_t)g.splits * g.n_tail * kPair * kTM;
}
int64_t ws_bytes_of(const PrefixGeom& g) {
  return tail_rows(g) * (tile_dim(g.d) * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
}

// Everything of a call but its sizes.
struct PrefixCall {
  const void *q, *k, *v;        // queries; prefix
  const void *own_k, *own_v;    // own tokens or NULL
  Strides3 sk, sv;              // their strides
  PrefixOut out;
  float scale;
  void* ws;
  const QAttend* beside;        // a cache's attend call that runs beside the prefix, or NULL
  cudaStream_t stream;
};

template <typename T, int D, int STAGES>
int launch_prefix(const PrefixCall& c, const PrefixGeom& geo) {
  using L = PrefixLayout<D, STAGES>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mk, mv, mok, mov;
  const uint64_t d = (uint64_t)geo.d, P = (uint64_t)geo.P, h = (uint64_t)geo.kv_heads;
  const int64_t head = (int64_t)geo.P * geo.d;
  const Strides3 st{geo.kv_heads * head, head, geo.d};
  if (int rc = make_tmap_4d(&mk, c.k, kBF16, d, P, h, 1, st, kTN)) return rc;
  if (int rc = make_tmap_4d(&mv, c.v, kBF16, d, P, h, 1, st, kTN)) return rc;
  mok = mk;
  mov = mv;
  if (geo.own) {
    const uint64_t n = (uint64_t)geo.n_q, b = (uint64_t)geo.batch;
    if (int rc = make_tmap_4d(&mok, c.own_k, kBF16, d, n, h, b, c.sk, (uint32_t)geo.box)) return rc;
    if (int rc = make_tmap_4d(&mov, c.own_v, kBF16, d, n, h, b, c.sv, (uint32_t)geo.box)) return rc;
  }
  PrefixOut out = c.out;
  out.stats = (float2*)c.ws;   // tail_rows is a multiple of 256, so part stays aligned
  out.part = (float*)((char*)c.ws + tail_rows(geo) * (int64_t)sizeof(float2));
  auto kern = prefix_tc_kernel<T, D, STAGES>;
  static std::atomic<uint64_t> ready{0};
  if (int rc = once_per_device(ready, [&] {
        return check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)L::kAlloc),
                          "cudaFuncSetAttribute(prefix_tc)");
      }))
    return rc;
  {
    LaunchScope ls("prefix_tc_kernel", c.stream);
    kern<<<(unsigned)(geo.n_full + geo.n_tail * geo.splits), kThreads, L::kAlloc, c.stream>>>(
        (const T*)c.q, mk, mv, mok, mov, out, c.scale * kLog2e, geo, device_status_ptr());
  }
  if (int rc = check_launch("prefix_tc_kernel")) return rc;
  if (c.beside != nullptr)
    if (int rc = qcache_attend_launch(*c.beside)) return rc;
  if (geo.n_tail == 0) return SBFA_OK;
  const int64_t rows_per = kMergeThreads / (D / 4);
  const int64_t blocks = ((int64_t)geo.n_tail * kPair * kTM + rows_per - 1) / rows_per;
  LaunchScope ls("prefix_merge_kernel", c.stream);
  return check_cuda(launch_early(prefix_merge_kernel<T, D>, (unsigned)blocks, kMergeThreads, 0,
                                 c.stream, true, out, geo),
                    "prefix_merge_kernel");
}

// Checks what the entry points share; launches behind it.
int check_call(PrefixCall& c, const int64_t* q_strides, PrefixGeom& geo, int64_t H,
               double softmax_scale, int64_t ws_bytes) {
  if (!(softmax_scale > 0) || softmax_scale > 1e30)
    return fail(SBFA_ERR_INVALID, "softmax_scale must be positive and finite");
  if (!c.q || !c.k || !c.v || !c.out.o)
    return fail(SBFA_ERR_INVALID, "prefix attention: NULL tensor pointer");
  geo.sn = q_strides ? q_strides[2] : geo.d;
  geo.sh = q_strides ? q_strides[1] : (int64_t)geo.n_q * geo.d;
  geo.sb = q_strides ? q_strides[0] : H * geo.n_q * geo.d;
  if (geo.sb < 0 || geo.sh < 0 || geo.sn < 0 || geo.sb % 8 || geo.sh % 8 || geo.sn % 8)
    return fail(SBFA_ERR_INVALID,
                "prefix attention: q strides must be non-negative multiples of 8 elements");
  for (const void* p : {c.q, c.k, c.v, c.out.own_o, (const void*)c.out.o, (const void*)c.ws})
    if ((uintptr_t)p & 15u)
      return fail(SBFA_ERR_INVALID, "prefix attention: tensors must be 16-byte aligned");
  const int64_t need = ws_bytes_of(geo);
  if (need > 0 && (c.ws == nullptr || ws_bytes < need))
    return fail(SBFA_ERR_INVALID, "prefix attention: workspace too small (need " +
                                      std::to_string(need) + " bytes)");
  c.scale = (float)softmax_scale;
  return SBFA_OK;
}

int launch_call(const PrefixCall& c, const PrefixGeom& geo, int dtype) {
  if (tile_dim(geo.d) == 64)
    return dtype == SBFA_BF16 ? launch_prefix<__nv_bfloat16, 64, 8>(c, geo)
                              : launch_prefix<__half, 64, 8>(c, geo);
  return dtype == SBFA_BF16 ? launch_prefix<__nv_bfloat16, 128, 5>(c, geo)
                            : launch_prefix<__half, 128, 5>(c, geo);
}

int check_prefix(int64_t B, int64_t H, int64_t kv_heads, int64_t n_q, int64_t P, int64_t head_dim,
                 int dtype, int64_t window, PrefixGeom* geo, const sbfa_qcache* cache = nullptr) {
  if (dtype != SBFA_F16 && dtype != SBFA_BF16)
    return fail(SBFA_ERR_UNSUPPORTED, "prefix attention: dtype must be float16 or bfloat16");
  if (tile_dim(head_dim) == 0)
    return fail(SBFA_ERR_UNSUPPORTED,
                "prefix attention: head_dim must be a multiple of 8 and at most 128");
  if (!prefix_geometry(B, H, kv_heads, n_q, P, head_dim, window, geo, cache))
    return fail(SBFA_ERR_INVALID, "prefix attention: sizes must be positive, H a multiple of "
                                  "kv_heads, P and B * H / kv_heads * n_q below 2^31");
  return SBFA_OK;
}

// SMs that the prefix's kernel holds for most of its time: none when it comes in several waves,
// behind whose last the cache's kernel starts.
int busy_sms(const PrefixGeom& g) {
  const int64_t ctas = (int64_t)g.n_tail * g.splits;
  return ctas < device_sm_count() ? (int)ctas : 0;
}

int64_t own_bytes(int64_t B, int64_t H, int64_t d) {
  return (B * H * (d + 1) * (int64_t)sizeof(float) + 255) / 256 * 256;
}

}  // namespace
}  // namespace sbfa

using namespace sbfa;

extern "C" int64_t sbfa_prefix_workspace_bytes(int64_t B, int64_t H, int64_t kv_heads,
                                               int64_t n_q, int64_t P, int64_t head_dim,
                                               int64_t window) {
  PrefixGeom geo;
  if (!prefix_geometry(B, H, kv_heads, n_q, P, head_dim, window, &geo)) return -1;
  return ws_bytes_of(geo);
}

extern "C" int sbfa_prefix_attend(const void* q, const int64_t* q_strides, const void* k_prefix,
                                  const void* v_prefix, const void* own_o, const float* own_lse,
                                  void* o, float* lse, int64_t B, int64_t H, int64_t kv_heads,
                                  int64_t n_q, int64_t P, int64_t head_dim, int dtype,
                                  double softmax_scale, void* ws, int64_t ws_bytes,
                                  void* stream) {
  PrefixGeom geo;
  if (int rc = check_prefix(B, H, kv_heads, n_q, P, head_dim, dtype, 0, &geo)) return rc;
  if ((own_o == nullptr) != (own_lse == nullptr))
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_attend: own_o and own_lse come together");
  PrefixCall c = {};
  c.q = q;
  c.k = k_prefix;
  c.v = v_prefix;
  c.out.o = o;
  c.out.lse = lse;
  c.out.own_o = own_o;
  c.out.own_lse = own_lse;
  c.out.own_kind = own_o ? kOwn16 : kOwnNone;
  c.ws = ws;
  c.stream = (cudaStream_t)stream;
  if (int rc = check_call(c, q_strides, geo, H, softmax_scale, ws_bytes)) return rc;
  return launch_call(c, geo, dtype);
}

extern "C" int64_t sbfa_qcache_prefix_workspace_bytes(const sbfa_qcache* cache, int64_t H,
                                                      int64_t P) {
  PrefixGeom geo;
  if (qcache_attend_ws_bytes(cache, H, 0) < 0 ||   // refuses what is no cache
      !prefix_geometry(cache->batch, H, cache->kv_heads, 1, P, cache->head_dim, 0, &geo, cache))
    return -1;
  const int64_t bytes = qcache_attend_ws_bytes(cache, H, busy_sms(geo));
  return own_bytes(cache->batch, H, cache->head_dim) + ws_bytes_of(geo) + bytes;
}

extern "C" int sbfa_qcache_prefix_attend(const sbfa_qcache* cache, const void* q,
                                         const void* k_prefix, const void* v_prefix, int64_t P,
                                         void* o, float* lse, int64_t H, double softmax_scale,
                                         void* ws, int64_t ws_bytes, void* stream) {
  if (cache == nullptr) return fail(SBFA_ERR_INVALID, "8-bit cache: NULL cache");
  const int64_t B = cache->batch, head_dim = cache->head_dim;
  PrefixGeom geo;
  if (int rc = check_prefix(B, H, cache->kv_heads, 1, P, head_dim, cache->dtype, 0, &geo, cache))
    return rc;
  // the cache's own result in fp32 [B, H, d] and its LSE [B, H], the prefix's scratch, the cache's
  const int64_t own = own_bytes(B, H, head_dim), pre = ws_bytes_of(geo);
  if (ws == nullptr || ws_bytes < own + pre)
    return fail(SBFA_ERR_INVALID, "sbfa_qcache_prefix_attend: workspace too small");
  float* own_o = (float*)ws;
  float* own_lse = own_o + B * H * head_dim;
  const QAttend a{cache, q, nullptr, own_o, own_lse, H, softmax_scale, (char*)ws + own + pre,
                  ws_bytes - own - pre, true, busy_sms(geo), (cudaStream_t)stream};
  PrefixCall c = {};
  c.q = q;
  c.k = k_prefix;
  c.v = v_prefix;
  c.out.o = o;
  c.out.lse = lse;
  c.out.own_o = own_o;
  c.out.own_lse = own_lse;
  c.out.own_kind = kOwn32;
  c.ws = (char*)ws + own;
  c.beside = &a;
  c.stream = (cudaStream_t)stream;
  // all checks before the first launch
  if (int rc = qcache_attend_check(a)) return rc;
  if (int rc = check_call(c, nullptr, geo, H, softmax_scale, pre)) return rc;
  return launch_call(c, geo, cache->dtype);
}

extern "C" int sbfa_prefix_prompt(const void* q, const void* k, const void* v,
                                  const int64_t* strides, const void* k_prefix,
                                  const void* v_prefix, void* o, float* lse, int64_t B, int64_t H,
                                  int64_t kv_heads, int64_t n_q, int64_t P, int64_t head_dim,
                                  int dtype, double softmax_scale, int64_t window, void* ws,
                                  int64_t ws_bytes, void* stream) {
  return sbfa_prefix_prompt_sinks(q, k, v, strides, k_prefix, v_prefix, o, lse, B, H, kv_heads, n_q,
                                  P, head_dim, dtype, softmax_scale, 0, window, ws, ws_bytes, stream);
}

extern "C" int sbfa_prefix_prompt_sinks(const void* q, const void* k, const void* v,
                                        const int64_t* strides, const void* k_prefix,
                                        const void* v_prefix, void* o, float* lse, int64_t B,
                                        int64_t H, int64_t kv_heads, int64_t n_q, int64_t P,
                                        int64_t head_dim, int dtype, double softmax_scale,
                                        int64_t sink, int64_t window, void* ws, int64_t ws_bytes,
                                        void* stream) {
  PrefixGeom geo;
  if (int rc = check_prefix(B, H, kv_heads, n_q, P, head_dim, dtype, window, &geo)) return rc;
  if (window < 1)
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_prompt: window must be at least 1");
  if (sink < 0) return fail(SBFA_ERR_INVALID, "sbfa_prefix_prompt: sink must not be negative");
  geo.sink = (int)std::min(sink, n_q);
  if (!k || !v) return fail(SBFA_ERR_INVALID, "sbfa_prefix_prompt: NULL tensor pointer");
  PrefixCall c = {};
  c.q = q;
  c.k = k_prefix;
  c.v = v_prefix;
  c.own_k = k;
  c.own_v = v;
  c.out.own_v = v;
  const int64_t hk = geo.kv_heads;
  const Strides3 dense{hk * n_q * head_dim, n_q * head_dim, head_dim};
  c.sk = strides ? Strides3{strides[3], strides[4], strides[5]} : dense;
  c.sv = strides ? Strides3{strides[6], strides[7], strides[8]} : dense;
  if (!tma_compatible(k, c.sk) || !tma_compatible(v, c.sv))
    return fail(SBFA_ERR_INVALID, "sbfa_prefix_prompt: k and v must be 16-byte aligned with "
                                  "strides that are positive multiples of 8 elements");
  c.out.sv = c.sv;
  c.out.o = o;
  c.out.lse = lse;
  c.ws = ws;
  c.stream = (cudaStream_t)stream;
  if (int rc = check_call(c, strides, geo, H, softmax_scale, ws_bytes)) return rc;
  return launch_call(c, geo, dtype);
}
